// tree_attn.cuh — what the two tree attention kernels (tree_attn.cu on mma.sync,
// tree_attn_tc.cu on tcgen05) share: arguments, splits, the cut of fp32 into bf16
// terms, and the way results leave a CTA.
#pragma once

#include <cuda.h>

#include "kernels.cuh"
#include "mma_sync.cuh"
#include "verify.cuh"

namespace dllm {

// Everything a CTA needs to know of its sequence travels as kernel arguments: a load
// from memory before the first K/V address is known would cost every CTA its latency.
struct TAKernelArgs {
  TreeAttnArgs a;
  int bps;                  // blocks per split
  int seq[kTreeMaxSeqs];
  int row0[kTreeMaxSeqs];
  int m[kTreeMaxSeqs];
  int t0[kTreeMaxSeqs];
  int part0[kTreeMaxSeqs];  // first partial row of a split sequence
};

DLLM_DEV TreeSeq ta_seq(const TAKernelArgs& P, int i) { return TreeSeq{P.seq[i], P.row0[i], P.m[i], 0}; }

// The number of splits of a sequence with `slots` slots; the same on host and device.
__host__ __device__ inline int ta_splits(int slots, int bn, int bps) {
  const int blocks = (slots + bn - 1) / bn;
  return (blocks + bps - 1) / bps;
}

// One row tile of a CTA: rows [r0, r0 + RT) of the m G rows that share a KV head.
struct TATile {
  TreeSeq sq;
  int G, inv_g, head, r0, R, nsplit, split;
  DLLM_DEV void set_group(int g) { G = g, inv_g = (65536 + g - 1) / g; }
  // row / G for rows below 2^13 (there are at most 64 nodes x 8 heads)
  DLLM_DEV int node_of(int r) const { return r * inv_g >> 16; }
};

// The results of WS slot groups, each with RT rows of [HD + 4] outputs in sO and (max,
// sum) in sML, to `out`, or to this split's partials. HD / 4 threads per row.
template <int HD, int WS, int RT, int THREADS>
DLLM_DEV void ta_finish(const TAKernelArgs& P, const TATile& k, const float* sO, const float* sML, int tid) {
  const TreeAttnArgs& a = P.a;
  constexpr int kLanes = HD / 4, kStep = THREADS / kLanes;
  const int d = (tid % kLanes) * 4, rows = min(RT, k.R - k.r0);
  const size_t split_base = (size_t)P.part0[blockIdx.z] + (size_t)k.split * k.sq.m * a.nq;
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
    const int r = k.r0 + row, node = k.node_of(r), at = node * a.nq + k.head * k.G + (r - node * k.G);
    if (k.nsplit == 1) {
      const float inv = 1.0f / l;
      *reinterpret_cast<float4*>(a.out + ((size_t)k.sq.row0 * a.nq + at) * HD + d) =
          make_float4(f.x * inv, f.y * inv, f.z * inv, f.w * inv);
    } else {
      *reinterpret_cast<float4*>(a.part_o + (split_base + at) * HD + d) = f;
      if (d == 0) *reinterpret_cast<float2*>(a.part_ml + (split_base + at) * 2) = make_float2(m, l);
    }
  }
}

// tree_attn_tc.cu (bf16 caches), tree_attn_tc32.cu (fp32 caches)
constexpr int kTcBlock = 64;   // slots per block
constexpr int kTcRows = 128;   // rows per tile
cudaError_t configure_tree_attn_tc();
cudaError_t launch_tree_attn_tc(const TAKernelArgs& P, int hd, dim3 grid, cudaStream_t st);
cudaError_t configure_tree_attn_tc32();
cudaError_t launch_tree_attn_tc32(const TAKernelArgs& P, int hd, dim3 grid, cudaStream_t st);

}  // namespace dllm
