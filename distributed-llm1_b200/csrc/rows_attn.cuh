// rows_attn.cuh — attention of a batch of rows over a paged cache of fp32, bf16 or 4-bit
// rows, under a sliding window and first slots that stay visible, and the cache of 4-bit
// rows itself. rows_attn.cu runs few rows per sequence on mma.sync, rows_attn_tc.cu
// chunks on tcgen05, kv4.cu fills and reads the caches.
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "common.cuh"
#include "mma_sync.cuh"

namespace dllm {

constexpr int kRowsMaxSeqs = 128;  // sequences per batch: their places travel as kernel arguments
constexpr int kErrRowsWait = 8;    // a tcgen05 kernel of rows_attn_tc.cu gave up waiting on an mbarrier
constexpr int kGroup4 = 32;        // dims of a 4-bit row that share a scale and a minimum

enum KvKind { kKvF32 = 0, kKvBf16 = 1, kKv4 = 2 };

// Bytes of one head's row, without and with 4-bit rows' (scale, minimum) pairs.
template <int KIND, int HD>
struct KvRow {
  static constexpr int kBytes = KIND == kKvF32 ? HD * 4 : KIND == kKvBf16 ? HD * 2 : HD / 2;
  static constexpr int kPairs = KIND == kKv4 ? HD / kGroup4 : 0;  // u32 each: bf16 scale low, bf16 minimum high
};

// A paged cache as rows: row (page, head, offset) of a layer is number (page * kvh + head) *
// page_size + offset. KvLayout says the same in elements.
struct RowPages {
  const int* table;  // [sequences][max_pages]
  int log2_page, max_pages, kvh;
  DLLM_DEV size_t row(int seq, int slot, int head) const {
    const int phys = table[(size_t)seq * max_pages + (slot >> log2_page)];
    return (((size_t)phys * kvh + head) << log2_page) + (slot & ((1 << log2_page) - 1));
  }
};

// The rows of a batch: row j of sequence i is batch row row0[i] + j and cache slot t0[i] + j.
struct RowsBatch {
  int n_seqs;
  int seq[kRowsMaxSeqs];
  int row0[kRowsMaxSeqs];
  int m[kRowsMaxSeqs];
  int t0[kRowsMaxSeqs];
};

struct RowsAttnArgs {
  const float* q;  // [n][nq][hd]
  float* out;      // [n][nq][hd]
  const void *kc, *vc;       // the layer's rows
  const uint32_t *ks, *vs;   // 4-bit rows: their (scale, minimum) pairs
  RowPages pages;
  int nq;
  int window, sinks;         // row at slot p sees s <= p where s > p - window or s < sinks
  float scale_log2;          // log2(e) / sqrt(hd)
  int* err;
  void* planes;              // scratch for the K and V blocks of long chunks in fp16 (rows_attn_tc.cu)
  size_t planes_bytes;
  unsigned char* exps;       // in it: exponents of the powers of two per slot (set by op_rows_attention),
  uint16_t* info;            // and the blocks' exponents and flags
  float* part_o;             // [rows][hd] partial outputs of sequences that are split
  float* part_ml;            // [rows][2]
};
size_t rows_attn_part_rows(int sms);  // capacity of part_o / part_ml
// The scratch a call wants: all its long chunks at once, but no more than 1 GB unless one
// sequence needs it (the others take turns then).
size_t rows_attn_planes_bytes(const RowsAttnArgs& a, const RowsBatch& b, int kind, int hd);
cudaError_t configure_rows_attn();
cudaError_t op_rows_attention(const RowsAttnArgs& a, const RowsBatch& b, int kind, int hd, int sms, int* launches,
                              cudaStream_t st);

// ---- kv4.cu: fp32 rows [n][kvh][hd] -> slots t0 + j, and 4-bit rows back
cudaError_t op_rows_append(const RowsBatch& b, int n, const RowPages& p, int kind, int hd, const float* k, const float* v,
                           void* kc, void* vc, uint32_t* ks, uint32_t* vs, cudaStream_t st);
cudaError_t op_rows_read4(const RowsBatch& b, int n, const RowPages& p, int hd, const void* kc, const void* vc,
                          const uint32_t* ks, const uint32_t* vs, float* k, float* v, cudaStream_t st);

// ---- what the attention kernels share --------------------------------------------------

// The blocks of bn slots that rows of a sequence need, for rows at slots p0..p1: those of the
// sinks, then those from the first slot that p0 sees to p1. Block b of them starts at slot
// slot0(b).
struct RowsView {
  int p0, p1, nsink, first, nb;
  __host__ __device__ RowsView(int p0_, int p1_, int window, int sinks, int bn) : p0(p0_), p1(p1_) {
    const int lo = p0 + 1 > window ? p0 + 1 - window : 0;
    first = lo / bn;
    const int s = ((sinks < lo ? sinks : lo) + bn - 1) / bn;
    nsink = s < first ? s : first;
    nb = nsink + p1 / bn + 1 - first;
  }
  DLLM_DEV int slot0(int b, int bn) const { return (b < nsink ? b : b - nsink + first) * bn; }
  // Whether some row sees only a part of the bn slots from s0 on.
  DLLM_DEV bool edge(int s0, int bn, int window, int sinks) const {
    return s0 + bn - 1 > p0 || (s0 <= p1 - window && s0 + bn > sinks);
  }
};
DLLM_DEV bool rows_sees(int p, int s, int window, int sinks) { return s <= p && (s > p - window || s < sinks); }

// All tiles of rt rows of a batch (sequence by sequence, KV head by KV head), and their blocks one
// after the other, cut into a share per CTA: CTA c takes count[c] blocks from block begin_block[c]
// of tile begin_tile[c] on. A tile in one CTA's share is written out; of the others each CTA leaves
// partial results, at most two of rt rows (its first segment's, and its last one's), which are
// joined.
constexpr int kRowsMaxCtas = 320;
struct RowsKernelArgs {
  RowsAttnArgs a;
  int n_seqs;
  int seq[kRowsMaxSeqs], row0[kRowsMaxSeqs], m[kRowsMaxSeqs], t0[kRowsMaxSeqs];
  int tile0[kRowsMaxSeqs + 1];  // tiles before the sequence
  int unit0[kRowsMaxSeqs + 1];  // (KV head, block) pairs before the sequence (rows_attn_tc.cu)
  int begin_tile[kRowsMaxCtas], begin_block[kRowsMaxCtas], count[kRowsMaxCtas];
  int split_tile[kRowsMaxCtas], split_cta[kRowsMaxCtas], split_n[kRowsMaxCtas];  // joined tiles, their first CTA, CTAs
};
static_assert(sizeof(RowsKernelArgs) <= 16384, "kernel arguments");

DLLM_DEV int rows_find(const int* first, int n, int item) {
  int lo = 0, hi = n;  // first[lo] <= item < first[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (first[mid] <= item) lo = mid;
    else hi = mid;
  }
  return lo;
}

// One tile: rows [r0, r0 + rt) of the R = m G rows of a sequence that share a KV head (row r is query
// head r % G of batch row r / G).
struct RowsTile {
  int i, seq, row0, m, t0, head, G, r0, R;
  RowsView v;
  __host__ __device__ static int tiles_of(int m, int G, int rt) { return (m * G + rt - 1) / rt; }
  DLLM_DEV RowsTile(const RowsKernelArgs& P, int tile, int rt, int bn) : v(0, 0, 1, 0, 1) {
    i = rows_find(P.tile0, P.n_seqs, tile);
    seq = P.seq[i], row0 = P.row0[i], m = P.m[i], t0 = P.t0[i];
    G = P.a.nq / P.a.pages.kvh, R = m * G;
    const int tiles = tiles_of(m, G, rt), at = tile - P.tile0[i];
    head = at / tiles;
    r0 = at % tiles * rt;
    const int last = (r0 + rt < R ? r0 + rt : R) - 1;
    v = RowsView(t0 + r0 / G, t0 + last / G, P.a.window, P.a.sinks, bn);
  }
  // cache slot of row r, or -1 behind the last row
  DLLM_DEV int slot_of(int r) const { return r < R ? t0 + r / G : -1; }
  // (batch row within the sequence, query head) of row r as one number
  DLLM_DEV int place(int r, int nq) const { return r / G * nq + head * G + r % G; }
};

// One CTA's segments: calls f(tile, its first block, the block behind its last one, whether it is
// the CTA's first).
template <typename F>
DLLM_DEV void rows_segments(const RowsKernelArgs& P, int rt, int bn, F f) {
  int tile = P.begin_tile[blockIdx.x], b0 = P.begin_block[blockIdx.x];
  int left = P.count[blockIdx.x];
  for (bool first = true; left > 0; first = false) {
    const RowsTile k(P, tile, rt, bn);
    const int b1 = min(k.v.nb, b0 + left);
    f(k, b0, b1, first);
    left -= b1 - b0;
    ++tile, b0 = 0;
  }
}

// Cuts a batch into shares for at most max_ctas CTAs, none of less than `least` blocks unless there
// are fewer: equal shares of all blocks, or, where that is no slower, shares that end with their
// tiles (a CTA's second segment costs it a start, about as long as `start` blocks).
struct RowsPlan {
  int ctas, splits, most_n, units;  // CTAs, joined tiles, the most segments of one, (KV head, block) pairs
};
RowsPlan rows_plan(const RowsAttnArgs& a, const RowsBatch& b, int rt, int bn, int max_ctas, int least, int start, RowsKernelArgs* P);
// Joins the split tiles' segments.
cudaError_t rows_join(const RowsKernelArgs& P, const RowsPlan& plan, int rt, int bn, int hd, int* launches, cudaStream_t st);

// The results of WS slot groups, each with RT rows of [HD + 4] outputs in sO and (max, sum) in
// sML, to `out`, or where `whole` is false to the partial rows from `part` on. HD / 4 threads per
// row.
template <int HD, int WS, int RT, int THREADS>
DLLM_DEV void rows_finish(const RowsAttnArgs& a, const RowsTile& k, bool whole, size_t part, const float* sO, const float* sML,
                          int tid) {
  constexpr int kLanes = HD / 4, kStep = THREADS / kLanes;
  const int d = (tid % kLanes) * 4, rows = min(RT, k.R - k.r0);
#pragma unroll 4
  for (int row = tid / kLanes; row < rows; row += kStep) {
    float m = -INFINITY, l = 0.f;
#pragma unroll
    for (int w = 0; w < WS; ++w) m = fmaxf(m, sML[(w * RT + row) * 2]);
    const float base = m == -INFINITY ? 0.f : m;
    float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < WS; ++w) {
      const float e = WS == 1 ? 1.f : ex2(sML[(w * RT + row) * 2] - base);
      const float4 v = *reinterpret_cast<const float4*>(sO + (w * RT + row) * (HD + 4) + d);
      f.x = fmaf(v.x, e, f.x), f.y = fmaf(v.y, e, f.y), f.z = fmaf(v.z, e, f.z), f.w = fmaf(v.w, e, f.w);
      l = fmaf(sML[(w * RT + row) * 2 + 1], e, l);
    }
    if (whole) {
      const float inv = 1.0f / l;
      *reinterpret_cast<float4*>(a.out + ((size_t)k.row0 * a.nq + k.place(k.r0 + row, a.nq)) * HD + d) =
          make_float4(f.x * inv, f.y * inv, f.z * inv, f.w * inv);
    } else {
      *reinterpret_cast<float4*>(a.part_o + (part + row) * HD + d) = f;
      if (d == 0) *reinterpret_cast<float2*>(a.part_ml + (part + row) * 2) = make_float2(m, l);
    }
  }
}

}  // namespace dllm
