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
  void* info;                // in it: the blocks' factors (set by op_rows_attention)
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

// One kernel's share of a batch: its sequences, cut into CTAs. Item i of the grid belongs to
// the sequence whose [item0, item0 of the next) holds it.
struct RowsKernelArgs {
  RowsAttnArgs a;
  int n_seqs;
  int bps;  // blocks per split
  int seq[kRowsMaxSeqs], row0[kRowsMaxSeqs], m[kRowsMaxSeqs], t0[kRowsMaxSeqs];
  int item0[kRowsMaxSeqs + 1];   // CTAs: tiles (the last first), KV heads, splits
  int splits[kRowsMaxSeqs];      // of the sequence's tile that has most
  int part0[kRowsMaxSeqs];       // first partial row of a split sequence
  int join0[kRowsMaxSeqs + 1];   // joined (row, query head) pairs, 0 for sequences that are not split
};
static_assert(sizeof(RowsKernelArgs) <= 8192, "kernel arguments");

DLLM_DEV int rows_find(const int* first, int n, int item) {
  int lo = 0, hi = n;  // first[lo] <= item < first[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (first[mid] <= item) lo = mid;
    else hi = mid;
  }
  return lo;
}

// A CTA's work: rows [r0, r0 + rt) of the m G rows of a sequence that share a KV head (row r
// is query head r % G of batch row r / G), over the blocks [b0, b1) of their view.
struct RowsTile {
  int i, seq, row0, m, t0, head, G, r0, R, split, nsplit, b0, b1;
  RowsView v;
  DLLM_DEV RowsTile(const RowsKernelArgs& P, int item, int rt, int bn) : v(0, 0, 1, 0, 1) {
    i = rows_find(P.item0, P.n_seqs, item);
    seq = P.seq[i], row0 = P.row0[i], m = P.m[i], t0 = P.t0[i];
    const int kvh = P.a.pages.kvh;
    G = P.a.nq / kvh, R = m * G;
    const int at = item - P.item0[i], s = P.splits[i], tiles = (R + rt - 1) / rt;
    split = at % s;
    head = at / s % kvh;
    r0 = (tiles - 1 - at / s / kvh) * rt;
    const int last = (r0 + rt < R ? r0 + rt : R) - 1;
    v = RowsView(t0 + r0 / G, t0 + last / G, P.a.window, P.a.sinks, bn);
    nsplit = (v.nb + P.bps - 1) / P.bps;
    b0 = split * P.bps;
    b1 = b0 + P.bps < v.nb ? b0 + P.bps : v.nb;
  }
  // cache slot of row r, or -1 behind the last row
  DLLM_DEV int slot_of(int r) const { return r < R ? t0 + r / G : -1; }
  // (batch row within the sequence, query head) of row r as one number
  DLLM_DEV int place(int r, int nq) const { return r / G * nq + head * G + r % G; }
};

// The results of WS slot groups, each with RT rows of [HD + 4] outputs in sO and (max, sum) in
// sML, to `out`, or to this split's partials. HD / 4 threads per row.
template <int HD, int WS, int RT, int THREADS>
DLLM_DEV void rows_finish(const RowsKernelArgs& P, const RowsTile& k, const float* sO, const float* sML, int tid) {
  const RowsAttnArgs& a = P.a;
  constexpr int kLanes = HD / 4, kStep = THREADS / kLanes;
  const int d = (tid % kLanes) * 4, rows = min(RT, k.R - k.r0);
  const size_t split_base = (size_t)P.part0[k.i] + (size_t)k.split * k.m * a.nq;
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
    const int at = k.place(k.r0 + row, a.nq);
    if (k.nsplit == 1) {
      const float inv = 1.0f / l;
      *reinterpret_cast<float4*>(a.out + ((size_t)k.row0 * a.nq + at) * HD + d) =
          make_float4(f.x * inv, f.y * inv, f.z * inv, f.w * inv);
    } else {
      *reinterpret_cast<float4*>(a.part_o + (split_base + at) * HD + d) = f;
      if (d == 0) *reinterpret_cast<float2*>(a.part_ml + (split_base + at) * 2) = make_float2(m, l);
    }
  }
}

}  // namespace dllm
