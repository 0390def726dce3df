// tree_attn_tc.cuh — the pieces that the two tcgen05 tree attention kernels share (bf16
// caches in tree_attn_tc.cu, fp32 caches in tree_attn_tc32.cu).
#pragma once

#include "tc.cuh"
#include "tree_attn.cuh"

namespace dllm {

// q rows of the tile, scaled so that the softmax is in powers of two, as three bf16 planes
// (highest terms first) of swizzled 64-dim boxes, what the K-major descriptor reads.
// WORKERS threads, `me` the caller's number. Rows behind the last one stay as they are: a row
// of S, P and O comes from its row alone.
template <int HD, int WORKERS>
DLLM_DEV void ta_load_q(const TAKernelArgs& P, const TATile& k, unsigned char* sQ, int me) {
  constexpr int kTasks = kTcRows * HD / 8, kEach = (kTasks + WORKERS - 1) / WORKERS, kPlane = HD / 64 * kTcRows * 128;
  const TreeAttnArgs& a = P.a;
  float4 f[kEach], g[kEach];
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    const int i = me + e * WORKERS, row = i / (HD / 8), d = (i % (HD / 8)) * 8, r = k.r0 + row;
    if (i < kTasks && r < k.R) {
      const int node = k.node_of(r);
      const float* q = a.q + ((size_t)(k.sq.row0 + node) * a.nq + k.head * k.G + (r - node * k.G)) * HD + d;
      f[e] = *reinterpret_cast<const float4*>(q), g[e] = *reinterpret_cast<const float4*>(q + 4);
    }
  }
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    const int i = me + e * WORKERS, row = i / (HD / 8), d = (i % (HD / 8)) * 8;
    if (i >= kTasks || k.r0 + row >= k.R) break;
    uint4 h, m, l;
    const float c = a.scale_log2;
    split3(f[e].x * c, f[e].y * c, h.x, m.x, l.x);
    split3(f[e].z * c, f[e].w * c, h.y, m.y, l.y);
    split3(g[e].x * c, g[e].y * c, h.z, m.z, l.z);
    split3(g[e].z * c, g[e].w * c, h.w, m.w, l.w);
    unsigned char* at = sQ + (d / 64) * (kTcRows * 128) + row * 128 + ((((d % 64) >> 3) ^ (row & 7)) << 4);
    *reinterpret_cast<uint4*>(at) = h;
    *reinterpret_cast<uint4*>(at + kPlane) = m;
    *reinterpret_cast<uint4*>(at + 2 * kPlane) = l;
  }
}

// Which slots of a 64-slot block that starts at node `node0` (above -64; negative: in the
// context) a row with ancestors `anc` sees.
DLLM_DEV unsigned long long ta_sees(unsigned long long anc, int node0) {
  if (node0 >= 64) return 0ull;
  return node0 >= 0 ? anc >> node0 : (anc << -node0) | ((1ull << -node0) - 1);
}

// One block of the online softmax of one row: 64 scores in u0, u1 (as bits, overwritten). The
// row's running maximum m and sum l move on, p goes to tensor memory at `tp` as three planes
// of 32 columns of packed bf16 pairs, and the factor of the earlier output is returned. A row
// that has seen nothing keeps m = -inf, and every p is 0.
DLLM_DEV float ta_softmax_block(uint32_t (&u0)[32], uint32_t (&u1)[32], bool masked, unsigned long long see, float& m,
                                float& l, uint32_t tp) {
  if (masked) {
#pragma unroll
    for (int c = 0; c < 32; ++c) {
      if (!(see >> c & 1)) u0[c] = __float_as_uint(-INFINITY);
      if (!(see >> (c + 32) & 1)) u1[c] = __float_as_uint(-INFINITY);
    }
  }
  float x0 = m, x1 = -INFINITY, x2 = -INFINITY, x3 = -INFINITY;
#pragma unroll
  for (int c = 0; c < 32; c += 2) {
    x0 = fmaxf(x0, __uint_as_float(u0[c])), x1 = fmaxf(x1, __uint_as_float(u0[c + 1]));
    x2 = fmaxf(x2, __uint_as_float(u1[c])), x3 = fmaxf(x3, __uint_as_float(u1[c + 1]));
  }
  const float x = fmaxf(fmaxf(x0, x1), fmaxf(x2, x3)), b = x == -INFINITY ? 0.f : x, f = ex2(m - b);
  m = x;
  float s0 = 0.f, s1 = 0.f;
#pragma unroll
  for (int c = 0; c < 64; c += 16) {  // 8 packed columns of each plane at a time
    uint32_t ph[8], pm[8], pl[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float p0 = ex2(__uint_as_float(c < 32 ? u0[(c + 2 * e) & 31] : u1[(c + 2 * e) & 31]) - b);
      const float p1 = ex2(__uint_as_float(c < 32 ? u0[(c + 2 * e + 1) & 31] : u1[(c + 2 * e + 1) & 31]) - b);
      s0 += p0, s1 += p1;
      split3(p0, p1, ph[e], pm[e], pl[e]);
    }
    tmem_st8(tp + (uint32_t)(c / 2), ph);
    tmem_st8(tp + 32u + (uint32_t)(c / 2), pm);
    tmem_st8(tp + 64u + (uint32_t)(c / 2), pl);
  }
  l = fmaf(l, f, s0 + s1);
  return f;
}

// Adds the non-finite values of a block's drafted V rows where this row sees them (they were
// taken out of the operand, since 0 x NaN would reach every row).
template <typename KT, int HD>
DLLM_DEV void ta_add_nonfinite(const TAKernelArgs& P, const TATile& k, float (&o)[HD], unsigned long long see, int slot0, int T0) {
  for (int j = 0; j < kTcBlock; ++j) {
    const int slot = slot0 + j;
    if (slot < T0 || slot >= T0 + k.sq.m || !(see >> j & 1)) continue;
    const KT* v = static_cast<const KT*>(P.a.vc) + P.a.kv.offset(k.sq.seq, slot, k.head);
#pragma unroll
    for (int d = 0; d < HD; ++d) {
      float e;
      if constexpr (sizeof(KT) == 2) e = bf16_to_f32(v[d]);
      else e = v[d];
      if (!is_finite(e)) o[d] += e;
    }
  }
}

}  // namespace dllm
