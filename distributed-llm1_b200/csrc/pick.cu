// pick.cu — one token per row of logits under penalties for repeated tokens,
// additive biases and a grammar mask, and the processed logits where they are wanted.
//
// For token t of a row with logit x, c = occurrences among the generated tokens:
//   y = x > 0 ? x / repetition : x * repetition     if t occurs in the history at all
//   y = (y - frequency * c) - presence              if c > 0
//   y = y + bias[t]                                 if t is in the bias list
//   y = -inf                                        if the mask forbids t
// and the pick is the first allowed t with the largest y (NaN counts as -inf), -1
// where the mask allows nothing. Every step is one rounded 32-bit operation, as
// separate elementwise operations would round it. The history of a tree's node is
// its sequence's tokens, then the drafted tokens on the path from the root to it.
//
// Bound by memory: the logits are read once (and written once); history, biases
// and mask are small beside them. The vocabulary is cut into one slice per CTA of a
// cluster. A CTA counts the history's tokens that fall into its slice in shared
// memory (integer atomics, so their order does not matter), then streams its
// slice of kRows rows that share that history; a tree's row adds its own path's
// tokens before and takes them out after. The CTAs' best (value, index) keys meet in
// the first CTA's shared memory: no global scratch, nothing to reset, one launch.
#include <cooperative_groups.h>

#include "verify.cuh"

namespace cg = cooperative_groups;

namespace dllm {
namespace {

constexpr int kPickThreads = 512;
constexpr int kPickWarps = kPickThreads / 32;
constexpr int kMaxCluster = 16;
constexpr int kMaxChunk = 12288;  // tokens of a slice held in shared memory at a time
constexpr int kMaxRowsPerCta = 8;

constexpr uint32_t kGiven = 0x80000000u;  // the token occurs among the given (prompt) tokens

struct PickSmem {
  unsigned long long key[kMaxRowsPerCta][kMaxCluster];  // of the first CTA: every CTA's best
  unsigned long long warp_key[kMaxRowsPerCta][kPickWarps];
};

// Best allowed token so far of one thread, which sees tokens in ascending order.
struct Best {
  float v = -INFINITY;
  int t = -1;
  DLLM_DEV void see(float y, int tok) {
    if (t < 0 || y > v) {  // a NaN is never greater
      v = y == y ? y : -INFINITY;
      t = tok;
    }
  }
};

struct RowRules {
  float rep, freq, pres;
  const uint32_t* mask;     // the row's words or null
  const float* bias_val;    // of the row's sequence or null
};

// The rules above for one token. cnt: its count word; b: 1 + its entry in the bias
// list, or 0.
DLLM_DEV float apply(float x, uint32_t cnt, uint32_t b, const RowRules& r) {
  if (cnt) {
    x = x > 0.f ? __fdiv_rn(x, r.rep) : __fmul_rn(x, r.rep);
    const uint32_t c = cnt & ~kGiven;
    if (c) x = __fsub_rn(__fsub_rn(x, __fmul_rn(r.freq, (float)c)), r.pres);
  }
  if (b) x = __fadd_rn(x, r.bias_val[b - 1]);
  return x;
}

DLLM_DEV int clampi(int v, int lo, int hi) { return v < lo ? lo : (v > hi ? hi : v); }

// Grid: clusters of `csize` CTAs; cluster = (sequence, group of `rows` rows).
__global__ void __launch_bounds__(kPickThreads) pick_kernel(const PickArgs a, int rows, int groups, int slice, int chunk) {
  extern __shared__ __align__(16) uint32_t dyn[];  // counts [chunk], then bias entries [chunk]
  __shared__ PickSmem sm;
  cg::cluster_group cluster = cg::this_cluster();
  const int csize = cluster.num_blocks(), rank = cluster.block_rank();
  const int item = blockIdx.x / csize;
  const int s = item / groups, group = item - s * groups;
  // the sequence's rows that this cluster handles
  const int m = a.seqs ? a.seqs[s].m : 1;
  const int row0 = a.seqs ? a.seqs[s].row0 : s;
  const int r0 = group * rows, r1 = min(m, r0 + rows);
  if (r0 >= r1) return;  // the whole cluster leaves
  cluster.barrier_arrive();

  const bool counting = a.penalties != nullptr;
  uint32_t* cnt = dyn;
  uint32_t* bia = counting ? dyn + chunk : dyn;
  int h0 = 0, h1 = 0, given = 0;
  if (counting && a.hist) {
    h0 = clampi(a.hist_off[s], 0, a.hist_total);
    h1 = clampi(a.hist_off[s + 1], h0, a.hist_total);
    given = h0 + (a.prompt ? clampi(a.prompt[s], 0, h1 - h0) : 0);
  }
  int b0 = 0, b1 = 0;
  if (a.bias_tok) {
    b0 = clampi(a.bias_off[s], 0, a.bias_total);
    b1 = clampi(a.bias_off[s + 1], b0, a.bias_total);
  }
  RowRules r;
  r.rep = counting ? a.penalties[3 * s] : 1.f;
  r.freq = counting ? a.penalties[3 * s + 1] : 0.f;
  r.pres = counting ? a.penalties[3 * s + 2] : 0.f;
  r.bias_val = a.bias_tok ? a.bias_val + b0 : nullptr;
  const int words = (a.vocab + 31) / 32;
  const int v0 = rank * slice, v1 = min(a.vocab, v0 + slice);

  if (threadIdx.x < kMaxRowsPerCta * kPickWarps) sm.warp_key[threadIdx.x / kPickWarps][threadIdx.x % kPickWarps] = 0ull;
  for (int c0 = v0; c0 < v1; c0 += chunk) {
    const int n = min(chunk, v1 - c0);
    __syncthreads();  // the previous chunk's counts are done with
    if (counting || a.bias_tok) {
      const int fill = (counting ? chunk : 0) + (a.bias_tok ? chunk : 0);
      for (int i = threadIdx.x; i < fill / 4; i += kPickThreads) reinterpret_cast<uint4*>(dyn)[i] = make_uint4(0, 0, 0, 0);
      __syncthreads();
#pragma unroll 4
      for (int i = h0 + threadIdx.x; i < h1; i += kPickThreads) {
        const unsigned t = (unsigned)(a.hist[i] - c0);  // ids outside the vocabulary fall into no slice
        if (t < (unsigned)n) {
          if (i < given)
            atomicOr(cnt + t, kGiven);
          else
            atomicAdd(cnt + t, 1u);
        }
      }
      for (int i = b0 + threadIdx.x; i < b1; i += kPickThreads) {
        const unsigned t = (unsigned)(a.bias_tok[i] - c0);
        if (t < (unsigned)n) atomicMax(bia + t, (uint32_t)(i - b0 + 1));  // of a token listed twice the last entry
      }
      __syncthreads();
    }
#pragma unroll 1
    for (int q = r0; q < r1; ++q) {
      const int row = row0 + q;
      if (counting && a.seqs) {  // the drafted tokens on the way to this node
        const unsigned long long anc = a.anc[row];
        if (threadIdx.x < m && (anc >> threadIdx.x & 1)) {
          const unsigned t = (unsigned)(a.draft[row0 + threadIdx.x] - c0);
          if (t < (unsigned)n) atomicAdd(cnt + t, 1u);
        }
        __syncthreads();
      }
      r.mask = a.mask ? a.mask + (size_t)row * words : nullptr;
      const float* x = a.logits + (size_t)row * a.vocab + c0;
      float* y = a.out ? a.out + (size_t)row * a.vocab + c0 : nullptr;
      Best bst;
      // 16-byte groups start where the row's address allows them
      const int lead = min(n, (int)((4 - (((size_t)row * a.vocab + c0) & 3)) & 3));
      const int body = (n - lead) / 4;
      auto one = [&](int t) {
        float v = apply(x[t], counting ? cnt[t] : 0, a.bias_tok ? bia[t] : 0, r);
        const int tok = c0 + t;
        if (r.mask && !(r.mask[tok >> 5] >> (tok & 31) & 1))
          v = -INFINITY;
        else
          bst.see(v, tok);
        if (y) y[t] = v;
      };
      if (threadIdx.x < lead) one(threadIdx.x);
      for (int i = threadIdx.x; i < body; i += kPickThreads) {
        const int t = lead + 4 * i, tok = c0 + t;
        float4 f = __ldcs(reinterpret_cast<const float4*>(x + t));
        uint32_t k4[4] = {0, 0, 0, 0}, b4[4] = {0, 0, 0, 0};
        if (counting) {
          if (lead == 0) {
            const uint4 u = *reinterpret_cast<const uint4*>(cnt + t);
            k4[0] = u.x, k4[1] = u.y, k4[2] = u.z, k4[3] = u.w;
          } else {
            for (int e = 0; e < 4; ++e) k4[e] = cnt[t + e];
          }
        }
        if (a.bias_tok) {
          if (lead == 0) {
            const uint4 u = *reinterpret_cast<const uint4*>(bia + t);
            b4[0] = u.x, b4[1] = u.y, b4[2] = u.z, b4[3] = u.w;
          } else {
            for (int e = 0; e < 4; ++e) b4[e] = bia[t + e];
          }
        }
        uint32_t bits = 0xfu;
        if (r.mask) {
          const int w = tok >> 5, sh = tok & 31;
          bits = r.mask[w] >> sh;
          if (sh > 28) bits |= r.mask[w + 1] << (32 - sh);  // the group's last token lies in the next word
        }
        float v[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (k4[e] | b4[e]) v[e] = apply(v[e], k4[e], b4[e], r);
          if (bits >> e & 1)
            bst.see(v[e], tok + e);
          else
            v[e] = -INFINITY;
        }
        if (y) __stcs(reinterpret_cast<float4*>(y + t), make_float4(v[0], v[1], v[2], v[3]));
      }
      const int tail = lead + 4 * body;
      if (threadIdx.x < n - tail) one(tail + threadIdx.x);
      unsigned long long k = bst.t < 0 ? 0ull : argmax_key(bst.v, bst.t);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const unsigned long long other = __shfl_xor_sync(0xffffffffu, k, o);
        if (other > k) k = other;
      }
      if ((threadIdx.x & 31) == 0 && k > sm.warp_key[q - r0][threadIdx.x >> 5]) sm.warp_key[q - r0][threadIdx.x >> 5] = k;
      if (counting && a.seqs) {
        __syncthreads();
        const unsigned long long anc = a.anc[row];
        if (threadIdx.x < m && (anc >> threadIdx.x & 1)) {
          const unsigned t = (unsigned)(a.draft[row0 + threadIdx.x] - c0);
          if (t < (unsigned)n) atomicSub(cnt + t, 1u);
        }
        __syncthreads();
      }
    }
  }
  __syncthreads();
  cluster.barrier_wait();  // every CTA of the cluster runs: its shared memory may be written
  if (threadIdx.x < r1 - r0) {
    unsigned long long k = 0;
    for (int w = 0; w < kPickWarps; ++w) k = sm.warp_key[threadIdx.x][w] > k ? sm.warp_key[threadIdx.x][w] : k;
    PickSmem* first = cluster.map_shared_rank(&sm, 0);
    first->key[threadIdx.x][rank] = k;
  }
  cluster.sync();
  if (rank == 0 && threadIdx.x < r1 - r0) {
    unsigned long long k = 0;
    for (int w = 0; w < csize; ++w) k = sm.key[threadIdx.x][w] > k ? sm.key[threadIdx.x][w] : k;
    a.tokens[row0 + r0 + threadIdx.x] = k ? argmax_key_index(k) : -1;
  }
}

}  // namespace

cudaError_t configure_pick_kernels() {
  cudaError_t e = cudaFuncSetAttribute(pick_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 2 * kMaxChunk * 4);
  if (e == cudaSuccess) e = cudaFuncSetAttribute(pick_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  return e;
}

cudaError_t op_pick(const PickArgs& a, int sms, cudaStream_t st) {
  const int csize = kMaxCluster;
  // rows per CTA: sequences with many rows share the counting of their history
  int rows = 1;
  while (rows < kMaxRowsPerCta && rows < a.max_m && (long long)a.n * csize / rows > 2ll * sms) rows *= 2;
  const int groups = (a.max_m + rows - 1) / rows;
  int slice = (a.vocab + csize - 1) / csize;
  slice = (slice + 127) / 128 * 128;
  const int chunk = slice < kMaxChunk ? slice : kMaxChunk;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)a.n_seqs * groups * csize);
  cfg.blockDim = dim3(kPickThreads);
  cfg.dynamicSmemBytes = (size_t)chunk * 4 * ((a.penalties ? 1 : 0) + (a.bias_tok ? 1 : 0));
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = csize;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, pick_kernel, a, rows, groups, slice, chunk);
}

}  // namespace dllm
