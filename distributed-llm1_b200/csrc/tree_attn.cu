// tree_attn.cu — attention of a drafted tree over a stage's paged KV cache.
//
// Node i of a sequence with T0 cached slots sees the slots [0, T0) and slot T0 + j
// for every node j on the path from the root to i, itself included:
//   out_i = sum_j p_ij v_j,  p_ij = exp(q_i . k_j / sqrt(hd) - max_i) / sum_i
// The G query heads of a KV head and the m nodes make m G rows that share one pass
// over that head's K and V; the softmax runs online over blocks of slots, and a
// sequence's slots are split over CTAs whose partial results a second kernel joins.
//
// Precision. q, p and the outputs are fp32 like every activation here, and the
// products run on the tensor cores all the same: with a bf16 cache q and p are cut
// into three bf16 terms (8 + 8 + 8 bits; the products with bf16 K and V are exact),
// with an fp32 cache all four operands into two tf32 terms. q, K and V are cut (a
// rounded high term could overflow), so that a low term is up to 2^-10 of its operand
// and has its sign: the scores take all four products, since without low x low each
// would be short by up to 2^-20 of itself. p, at most 1, is rounded: p_low v_low has
// either sign, stays below 2^-21 of the product and is left out. The tensor core adds into its fp32 accumulator with
// truncation, so long chains would drift towards zero by 2^-24 per step: the large
// terms and the corrections have accumulators of their own, a block's p . V starts
// from zero, and the sum over blocks is a rounded fp32 add in registers.
//
// Work split. A CTA has 8 warps and takes 16 WR rows of one (sequence, KV head): WR
// warps side by side in rows, 8 / WR of them in slots, so that one node's G rows
// still keep 8 warps busy. K and V blocks come through a cp.async ring, and slots
// behind the sequence's last one are zero-filled, never read.
#include <algorithm>

#include "tree_attn.cuh"

namespace dllm {
namespace {

constexpr int kTAThreads = 256;
constexpr float kNegInf = -INFINITY;

DLLM_DEV uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
DLLM_DEV void cp16_zfill(uint32_t dst, const void* src, bool real) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(real ? 16 : 0) : "memory");
}
DLLM_DEV void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
DLLM_DEV void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
DLLM_DEV void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
DLLM_DEV void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
DLLM_DEV void mma_bf16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
DLLM_DEV void mma_tf32(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// x = hi + lo, hi with 11 bits, cut; lo, the other 13, is rounded to 11 (2^-22 of x).
DLLM_DEV void split_tf32(float x, uint32_t& hi, uint32_t& lo) {
  hi = __float_as_uint(x) & 0xffffe000u;
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(lo) : "f"(x - __uint_as_float(hi)));
}
// The same with hi rounded to nearest; not for values next to the largest number.
DLLM_DEV void split_tf32_near(float x, uint32_t& hi, uint32_t& lo) {
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(hi) : "f"(x));
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(lo) : "f"(x - __uint_as_float(hi)));
}

// Tile shapes. SN: slots of a block that one warp takes; BN: slots of a block.
// The ring depth is what fits beside the q tile in 227 KB.
template <typename KT, int HD, int WR>
struct MmaTile {
  static constexpr bool kF32 = sizeof(KT) == 4;
  static constexpr int WS = 8 / WR;                 // warps side by side in slots
  static constexpr int SN = kF32 ? 8 * WR : WR == 1 ? 16 : 32;
  static constexpr int BN = SN * WS;                // 64, or 128 for up to 32 rows of a bf16 cache
  static constexpr int RT = 16 * WR;                // rows of the tile
  static constexpr int kRowBytes = HD * (int)sizeof(KT);
  static constexpr int kChunks = kRowBytes / 16;    // 16-byte chunks per slot
  static constexpr int kTileBytes = BN * kRowBytes; // one of K, V
  static constexpr int kQBytes = RT * HD * (kF32 ? 4 : 6);
  static constexpr int kMergeBytes = WS > 1 ? WS * RT * (HD + 2) * 4 : 0;
  static constexpr int kRoom = 225 * 1024 - kQBytes;
  static constexpr int kFit = kRoom / (2 * kTileBytes);
  static constexpr int kStages = kFit > 4 ? 4 : kFit;
  static_assert(kStages >= 2, "the K/V ring needs two stages");
  static_assert(kMergeBytes <= kStages * 2 * kTileBytes, "the join of the slot groups reuses the ring");
  static constexpr int kSmem = kQBytes + kStages * 2 * kTileBytes;
};

template <typename KT, int HD, int WR>
__global__ void __launch_bounds__(kTAThreads, 1) tree_attn_kernel(const __grid_constant__ TAKernelArgs P) {
  using T = MmaTile<KT, HD, WR>;
  constexpr int SN = T::SN, BN = T::BN, WS = T::WS, RT = T::RT, NT = SN / 8, CH = T::kChunks, S = T::kStages;
  constexpr bool F32 = T::kF32;
  extern __shared__ __align__(1024) unsigned char smem[];
  const TreeAttnArgs& a = P.a;
  asm volatile("griddepcontrol.launch_dependents;");  // the join may be scheduled; it waits for this grid's end
  TATile k;
  k.sq = ta_seq(P, blockIdx.z);
  k.set_group(a.nq / a.kvh);
  const int head = k.head = blockIdx.y % a.kvh, r0 = k.r0 = blockIdx.y / a.kvh * RT, R = k.R = k.sq.m * k.G;
  const int T0 = P.t0[blockIdx.z], slots = T0 + k.sq.m, split = k.split = blockIdx.x;
  k.nsplit = ta_splits(slots, BN, P.bps);
  if (r0 >= R || split >= k.nsplit) return;
  const TreeSeq& sq = k.sq;
  const int nblk = (slots + BN - 1) / BN;
  const int blk0 = split * P.bps, blk1 = min(nblk, blk0 + P.bps);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int wr = warp % WR, ws = warp / WR;
  const int g = lane >> 2, t = lane & 3;
  unsigned char* sQ = smem;
  unsigned char* ring = smem + T::kQBytes;

  // ---- K/V blocks through the ring. A thread copies one 16-byte chunk of every
  // (256 / CH)-th slot; pages hold at least 32 slots, so a block has BN / 32 page
  // lookups at most, made one block ahead of the copies that need them.
  constexpr int kPass = kTAThreads / CH;  // slots per pass
  constexpr int kPages = BN / 32;
  const int cch = tid % CH, crow = tid / CH;
  const KT* kc = static_cast<const KT*>(a.kc) + (size_t)head * a.kv.head_stride;
  const KT* vc = static_cast<const KT*>(a.vc) + (size_t)head * a.kv.head_stride;
  const int* table = a.kv.page_table + (size_t)sq.seq * a.kv.max_pages;
  int page[kPages];
  auto lookup = [&](int blk) {
#pragma unroll
    for (int i = 0; i < kPages; ++i) page[i] = __ldg(table + (min(blk * BN + 32 * i, slots - 1) >> a.kv.log2_page));
  };
  auto copy = [&](int blk, int stage) {
    const uint32_t dk = smem_addr(ring + stage * 2 * T::kTileBytes), dv = dk + T::kTileBytes;
#pragma unroll
    for (int i = 0; i < BN / kPass; ++i) {
      const int row = crow + i * kPass;
      const int slot = blk * BN + row;
      int pg = page[0];
#pragma unroll
      for (int u = 1; u < kPages; ++u) pg = row >= 32 * u ? page[u] : pg;
      const long long off = (long long)pg * a.kv.page_stride +
                            (long long)(slot & ((1 << a.kv.log2_page) - 1)) * a.kv.row_stride + cch * (16 / (int)sizeof(KT));
      const uint32_t at = row * T::kRowBytes + ((cch ^ (row & 7)) << 4);
      const bool real = slot < slots;
      cp16_zfill(dk + at, real ? kc + off : kc, real);
      cp16_zfill(dv + at, real ? vc + off : vc, real);
    }
  };
  lookup(blk0);
#pragma unroll
  for (int s = 0; s < S - 1; ++s) {
    if (blk0 + s < blk1) {
      copy(blk0 + s, s);
      lookup(blk0 + s + 1);
    }
    cp_commit();
  }

  // ---- the q tile, scaled by log2(e) / sqrt(hd) so that the softmax is in powers of two
  for (int i = tid; i < RT * HD / 4; i += kTAThreads) {
    const int row = i / (HD / 4), d = (i % (HD / 4)) * 4;
    const int r = r0 + row;
    float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
    if (r < R) {
      const int node = k.node_of(r);
      f = *reinterpret_cast<const float4*>(a.q + ((size_t)(sq.row0 + node) * a.nq + head * k.G + (r - node * k.G)) * HD + d);
      f.x *= a.scale_log2, f.y *= a.scale_log2, f.z *= a.scale_log2, f.w *= a.scale_log2;
    }
    if constexpr (F32) {
      *reinterpret_cast<float4*>(sQ + row * HD * 4 + (((d >> 2) ^ (row & 7)) << 4)) = f;
    } else {
      uint32_t h[2], m[2], l[2];
      split3(f.x, f.y, h[0], m[0], l[0]);
      split3(f.z, f.w, h[1], m[1], l[1]);
      unsigned char* p = sQ + row * HD * 2 + (((d >> 3) ^ (row & 7)) << 4) + (d & 4) * 2;
      *reinterpret_cast<uint2*>(p) = make_uint2(h[0], h[1]);
      *reinterpret_cast<uint2*>(p + RT * HD * 2) = make_uint2(m[0], m[1]);
      *reinterpret_cast<uint2*>(p + 2 * RT * HD * 2) = make_uint2(l[0], l[1]);
    }
  }

  // this thread's two rows of the tile and their ancestor masks
  const int ra = wr * 16 + g, rb = ra + 8;
  const unsigned long long anc_a = r0 + ra < R ? a.anc[sq.row0 + k.node_of(r0 + ra)] : 0ull;
  const unsigned long long anc_b = r0 + rb < R ? a.anc[sq.row0 + k.node_of(r0 + rb)] : 0ull;

  float o[HD / 8][4];
#pragma unroll
  for (int i = 0; i < HD / 8; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[i][e] = 0.f;
  float ma = kNegInf, mb = kNegInf, la = 0.f, lb = 0.f;

  for (int blk = blk0; blk < blk1; ++blk) {
    cp_wait<S - 2>();
    __syncthreads();
    {
      const int next = blk + S - 1;
      if (next < blk1) {
        copy(next, (next - blk0) % S);
        lookup(next + 1);
      }
      cp_commit();
    }
    unsigned char* sK = ring + ((blk - blk0) % S) * 2 * T::kTileBytes;
    unsigned char* sV = sK + T::kTileBytes;
    const int wslot = ws * SN;  // first slot of this warp within the block

    // ---- scores
    float sh[NT][4], ss[NT][4];
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) sh[i][e] = ss[i][e] = 0.f;
    if constexpr (F32) {
      // a chain of accumulators per product: one that takes several is waited for (16
      // sequences x 2 nodes x 12 heads at 4000 slots 45 us with two chains for three
      // products and loops of four, 41 so with four products)
      float s1[NT][4], s2[NT][4];
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) s1[i][e] = s2[i][e] = 0.f;
#pragma unroll
      for (int ks = 0; ks < HD / 8; ++ks) {
        uint32_t qh[4], ql[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int row = wr * 16 + g + (e & 1) * 8, ch = ks * 2 + (e >> 1);
          split_tf32(*reinterpret_cast<const float*>(sQ + row * HD * 4 + ((ch ^ (row & 7)) << 4) + t * 4), qh[e], ql[e]);
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const int row = wslot + nt * 8 + g;
          uint32_t kh[2], kl[2];
#pragma unroll
          for (int e = 0; e < 2; ++e)
            split_tf32(*reinterpret_cast<const float*>(sK + row * T::kRowBytes + (((ks * 2 + e) ^ (row & 7)) << 4) + t * 4),
                       kh[e], kl[e]);
          mma_tf32(ss[nt], ql, kl[0], kl[1]);
          mma_tf32(sh[nt], qh, kh[0], kh[1]);
          mma_tf32(s1[nt], qh, kl[0], kl[1]);
          mma_tf32(s2[nt], ql, kh[0], kh[1]);
        }
      }
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) ss[i][e] += s1[i][e] + s2[i][e];
    } else {
      const int arow = wr * 16 + (lane & 15);
      const uint32_t qa = smem_addr(sQ) + arow * HD * 2;
      const int krow = (lane & 7) + ((lane >> 4) << 3);
#pragma unroll
      for (int ks = 0; ks < HD / 16; ++ks) {
        uint32_t qh[4], qm[4], ql[4];
        const uint32_t at = qa + (((2 * ks + (lane >> 4)) ^ (arow & 7)) << 4);
        ldsm4(qh, at);
        ldsm4(qm, at + RT * HD * 2);
        ldsm4(ql, at + 2 * RT * HD * 2);
#pragma unroll
        for (int np = 0; np < NT / 2; ++np) {
          const int row = wslot + np * 16 + krow;
          uint32_t k4[4];
          ldsm4(k4, smem_addr(sK) + row * T::kRowBytes + (((2 * ks + ((lane >> 3) & 1)) ^ (row & 7)) << 4));
          mma_bf16(sh[2 * np], qh, k4[0], k4[1]);
          mma_bf16(sh[2 * np + 1], qh, k4[2], k4[3]);
          mma_bf16(ss[2 * np], qm, k4[0], k4[1]);
          mma_bf16(ss[2 * np + 1], qm, k4[2], k4[3]);
          mma_bf16(ss[2 * np], ql, k4[0], k4[1]);
          mma_bf16(ss[2 * np + 1], ql, k4[2], k4[3]);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) sh[i][e] += ss[i][e];

    // ---- mask: only blocks that reach behind the context have anything to hide
    const bool drafted = (blk + 1) * BN > T0;
    if (drafted) {
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int node = blk * BN + wslot + i * 8 + 2 * t + (e & 1) - T0;
          const unsigned long long anc = e < 2 ? anc_a : anc_b;
          if (node >= 0 && (node >= kTreeMaxNodes || !(anc >> node & 1))) sh[i][e] = kNegInf;
        }
    }

    // ---- online softmax
    float xa = kNegInf, xb = kNegInf;
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      xa = fmaxf(xa, fmaxf(sh[i][0], sh[i][1]));
      xb = fmaxf(xb, fmaxf(sh[i][2], sh[i][3]));
    }
#pragma unroll
    for (int w = 1; w < 4; w <<= 1) {
      xa = fmaxf(xa, __shfl_xor_sync(0xffffffffu, xa, w));
      xb = fmaxf(xb, __shfl_xor_sync(0xffffffffu, xb, w));
    }
    xa = fmaxf(xa, ma), xb = fmaxf(xb, mb);
    // rows that have seen nothing yet keep a maximum of -inf; their p are exp2(-inf - 0) = 0
    const float ba = xa == kNegInf ? 0.f : xa, bb = xb == kNegInf ? 0.f : xb;
    float fa = ex2(ma - ba), fb = ex2(mb - bb);
    ma = xa, mb = xb;
    float sa = 0.f, sb = 0.f;
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      sh[i][0] = ex2(sh[i][0] - ba), sh[i][1] = ex2(sh[i][1] - ba);
      sh[i][2] = ex2(sh[i][2] - bb), sh[i][3] = ex2(sh[i][3] - bb);
      sa += sh[i][0] + sh[i][1];
      sb += sh[i][2] + sh[i][3];
    }
    la = la * fa + sa, lb = lb * fb + sb;

    // ---- a drafted row that some nodes do not see may hold infinities or NaN, and
    // 0 * NaN would reach the nodes that must not see it: such values are taken out
    // of the tile and added to the rows that do see them.
    if (drafted) {
      int bad = 0;
      for (int i = tid; i < BN * HD; i += kTAThreads) {
        const int row = i / HD, d = i % HD;
        if (blk * BN + row < T0) continue;
        const KT* p = reinterpret_cast<const KT*>(sV + row * T::kRowBytes +
                                                  (((d * (int)sizeof(KT) >> 4) ^ (row & 7)) << 4) + (d * sizeof(KT) & 15));
        float v;
        if constexpr (F32) v = *p;
        else v = bf16_to_f32(*p);
        bad |= !is_finite(v);
      }
      if (__syncthreads_or(bad)) {
#pragma unroll
        for (int i = 0; i < HD / 8; ++i) {
          o[i][0] *= fa, o[i][1] *= fa, o[i][2] *= fb, o[i][3] *= fb;
          for (int row = wslot; row < wslot + SN; ++row) {
            const int node = blk * BN + row - T0;
            if (node < 0 || node >= sq.m) continue;
            const int d = i * 8 + 2 * t;
            const KT* p = reinterpret_cast<const KT*>(
                sV + row * T::kRowBytes + (((d * (int)sizeof(KT) >> 4) ^ (row & 7)) << 4) + (d * sizeof(KT) & 15));
            float v0, v1;
            if constexpr (F32) v0 = p[0], v1 = p[1];
            else v0 = bf16_to_f32(p[0]), v1 = bf16_to_f32(p[1]);
            if (anc_a >> node & 1) {
              if (!is_finite(v0)) o[i][0] += v0;
              if (!is_finite(v1)) o[i][1] += v1;
            }
            if (anc_b >> node & 1) {
              if (!is_finite(v0)) o[i][2] += v0;
              if (!is_finite(v1)) o[i][3] += v1;
            }
          }
        }
        fa = fb = 1.f;
        __syncthreads();
        for (int i = tid; i < BN * HD; i += kTAThreads) {
          const int row = i / HD, d = i % HD;
          if (blk * BN + row < T0) continue;
          KT* p = reinterpret_cast<KT*>(sV + row * T::kRowBytes + (((d * (int)sizeof(KT) >> 4) ^ (row & 7)) << 4) +
                                        (d * sizeof(KT) & 15));
          float v;
          if constexpr (F32) v = *p;
          else v = bf16_to_f32(*p);
          if (!is_finite(v)) *p = KT(0.f);
        }
        __syncthreads();
      }
    }

    // ---- o = o * f + p . V, the block's product from a fresh accumulator
    if constexpr (F32) {
      uint32_t ph[NT][4], pl[NT][4];
#pragma unroll
      for (int j = 0; j < NT; ++j) {  // slots 2t, 2t + 1 of a group take the places t, t + 4 of the product
        split_tf32_near(sh[j][0], ph[j][0], pl[j][0]);
        split_tf32_near(sh[j][2], ph[j][1], pl[j][1]);
        split_tf32_near(sh[j][1], ph[j][2], pl[j][2]);
        split_tf32_near(sh[j][3], ph[j][3], pl[j][3]);
      }
#pragma unroll
      for (int i = 0; i < HD / 8; ++i) {
        float ch[4] = {0.f, 0.f, 0.f, 0.f}, cs[4] = {0.f, 0.f, 0.f, 0.f};
        const int d = i * 8 + g;
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          uint32_t vh[2], vl[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int row = wslot + j * 8 + 2 * t + e;
            split_tf32(*reinterpret_cast<const float*>(sV + row * T::kRowBytes + (((d >> 2) ^ (row & 7)) << 4) + (d & 3) * 4),
                       vh[e], vl[e]);
          }
          mma_tf32(ch, ph[j], vh[0], vh[1]);
          mma_tf32(cs, ph[j], vl[0], vl[1]);
          mma_tf32(cs, pl[j], vh[0], vh[1]);
        }
        o[i][0] = fmaf(o[i][0], fa, ch[0] + cs[0]);
        o[i][1] = fmaf(o[i][1], fa, ch[1] + cs[1]);
        o[i][2] = fmaf(o[i][2], fb, ch[2] + cs[2]);
        o[i][3] = fmaf(o[i][3], fb, ch[3] + cs[3]);
      }
    } else {
      constexpr int NK = SN / 16;
      uint32_t ph[NK][4], pm[NK][4], pl[NK][4];
#pragma unroll
      for (int j = 0; j < NK; ++j) {
        split3(sh[2 * j][0], sh[2 * j][1], ph[j][0], pm[j][0], pl[j][0]);
        split3(sh[2 * j][2], sh[2 * j][3], ph[j][1], pm[j][1], pl[j][1]);
        split3(sh[2 * j + 1][0], sh[2 * j + 1][1], ph[j][2], pm[j][2], pl[j][2]);
        split3(sh[2 * j + 1][2], sh[2 * j + 1][3], ph[j][3], pm[j][3], pl[j][3]);
      }
      const int vrow = (lane & 7) + (((lane >> 3) & 1) << 3);
#pragma unroll
      for (int np = 0; np < HD / 16; ++np) {
        float ch[2][4], cs[2][4];
#pragma unroll
        for (int e = 0; e < 4; ++e) ch[0][e] = ch[1][e] = cs[0][e] = cs[1][e] = 0.f;
#pragma unroll
        for (int j = 0; j < NK; ++j) {
          const int row = wslot + j * 16 + vrow;
          uint32_t v4[4];
          ldsm4t(v4, smem_addr(sV) + row * T::kRowBytes + (((2 * np + (lane >> 4)) ^ (row & 7)) << 4));
          mma_bf16(ch[0], ph[j], v4[0], v4[1]);
          mma_bf16(ch[1], ph[j], v4[2], v4[3]);
          mma_bf16(cs[0], pm[j], v4[0], v4[1]);
          mma_bf16(cs[1], pm[j], v4[2], v4[3]);
          mma_bf16(cs[0], pl[j], v4[0], v4[1]);
          mma_bf16(cs[1], pl[j], v4[2], v4[3]);
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          float(&oo)[4] = o[2 * np + u];
          oo[0] = fmaf(oo[0], fa, ch[u][0] + cs[u][0]);
          oo[1] = fmaf(oo[1], fa, ch[u][1] + cs[u][1]);
          oo[2] = fmaf(oo[2], fb, ch[u][2] + cs[u][2]);
          oo[3] = fmaf(oo[3], fb, ch[u][3] + cs[u][3]);
        }
      }
    }
  }
  cp_wait<0>();
#pragma unroll
  for (int w = 1; w < 4; w <<= 1) {
    la += __shfl_xor_sync(0xffffffffu, la, w);
    lb += __shfl_xor_sync(0xffffffffu, lb, w);
  }

  // ---- results
  __syncthreads();  // the ring is free
  // through shared memory: rows padded by 4 floats keep the quads' stores apart
  constexpr int kPad = HD + 4;
  float* sO = reinterpret_cast<float*>(ring);
  float* sML = sO + WS * RT * kPad;
  static_assert(WS * RT * (kPad + 2) * 4 <= S * 2 * T::kTileBytes, "the results pass through the ring");
#pragma unroll
  for (int i = 0; i < HD / 8; ++i) {
    *reinterpret_cast<float2*>(sO + (ws * RT + ra) * kPad + i * 8 + 2 * t) = make_float2(o[i][0], o[i][1]);
    *reinterpret_cast<float2*>(sO + (ws * RT + rb) * kPad + i * 8 + 2 * t) = make_float2(o[i][2], o[i][3]);
  }
  if (t == 0) {
    sML[(ws * RT + ra) * 2] = ma, sML[(ws * RT + ra) * 2 + 1] = la;
    sML[(ws * RT + rb) * 2] = mb, sML[(ws * RT + rb) * 2 + 1] = lb;
  }
  __syncthreads();
  ta_finish<HD, WS, RT, kTAThreads>(P, k, sO, sML, tid);
}

// Joins the splits of a sequence. W warps share one (row, query head): warp w folds the
// splits w, w + W, ... in order, then the warps' results are folded in order, so the
// sum does not depend on timing. Every split's maximum, sum and output are loaded
// together: the chain is one load per kBatch splits.
template <int HD, int W>
__global__ void __launch_bounds__(256) tree_join_kernel(const __grid_constant__ TAKernelArgs P, int bn) {
  constexpr int V = HD / 32, kBatch = 4;
  __shared__ float so[8][HD], sml[8][2];
  const TreeAttnArgs& a = P.a;
  const TreeSeq sq = ta_seq(P, blockIdx.y);
  const int nsplit = ta_splits(P.t0[blockIdx.y] + sq.m, bn, P.bps);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int item = blockIdx.x * (8 / W) + warp / W, w = warp % W;
  const bool live = nsplit > 1 && item < sq.m * a.nq;
  const size_t step = (size_t)sq.m * a.nq, base = (size_t)P.part0[blockIdx.y] + item;
  asm volatile("griddepcontrol.wait;" ::: "memory");  // the splits' grid has ended and its stores are visible
  float m = kNegInf, l = 0.f, acc[V];
#pragma unroll
  for (int e = 0; e < V; ++e) acc[e] = 0.f;
  if (live) {
    for (int s0 = w; s0 < nsplit; s0 += kBatch * W) {
      float2 ml[kBatch];
      float o[kBatch][V];
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const int s = s0 + u * W;
        ml[u] = make_float2(kNegInf, 0.f);
#pragma unroll
        for (int e = 0; e < V; ++e) o[u][e] = 0.f;
        if (s < nsplit) {
          const size_t at = base + s * step;
          ml[u] = *reinterpret_cast<const float2*>(a.part_ml + at * 2);
          if constexpr (V == 4) {
            const float4 f = *reinterpret_cast<const float4*>(a.part_o + at * HD + lane * 4);
            o[u][0] = f.x, o[u][1] = f.y, o[u][2] = f.z, o[u][3] = f.w;
          } else {
            const float2 f = *reinterpret_cast<const float2*>(a.part_o + at * HD + lane * 2);
            o[u][0] = f.x, o[u][1] = f.y;
          }
        }
      }
      float x = m;
#pragma unroll
      for (int u = 0; u < kBatch; ++u) x = fmaxf(x, ml[u].x);
      const float b = x == kNegInf ? 0.f : x, f = ex2(m - b);
      m = x, l *= f;
#pragma unroll
      for (int e = 0; e < V; ++e) acc[e] *= f;
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const float wt = ex2(ml[u].x - b);
        l = fmaf(ml[u].y, wt, l);
#pragma unroll
        for (int e = 0; e < V; ++e) acc[e] = fmaf(o[u][e], wt, acc[e]);
      }
    }
  }
  if constexpr (W > 1) {
#pragma unroll
    for (int e = 0; e < V; ++e) so[warp][lane * V + e] = acc[e];
    if (lane == 0) sml[warp][0] = m, sml[warp][1] = l;
    __syncthreads();
    if (w != 0) return;
    float x = kNegInf;
#pragma unroll
    for (int u = 0; u < W; ++u) x = fmaxf(x, sml[warp + u][0]);
    const float b = x == kNegInf ? 0.f : x;
    l = 0.f;
#pragma unroll
    for (int e = 0; e < V; ++e) acc[e] = 0.f;
#pragma unroll
    for (int u = 0; u < W; ++u) {
      const float wt = ex2(sml[warp + u][0] - b);
      l = fmaf(sml[warp + u][1], wt, l);
#pragma unroll
      for (int e = 0; e < V; ++e) acc[e] = fmaf(so[warp + u][lane * V + e], wt, acc[e]);
    }
  }
  if (!live) return;
  const float inv = 1.0f / l;
  float* dst = a.out + ((size_t)sq.row0 * a.nq + item) * HD + lane * V;
#pragma unroll
  for (int e = 0; e < V; ++e) dst[e] = acc[e] * inv;
}

template <typename KT, int HD, int WR>
cudaError_t configure_one() {
  return cudaFuncSetAttribute(tree_attn_kernel<KT, HD, WR>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                              MmaTile<KT, HD, WR>::kSmem);
}
template <int HD>
cudaError_t configure_hd() {
  cudaError_t e = configure_one<float, HD, 1>();
  if (e == cudaSuccess) e = configure_one<float, HD, 2>();
  if (e == cudaSuccess) e = configure_one<__nv_bfloat16, HD, 1>();
  if (e == cudaSuccess) e = configure_one<__nv_bfloat16, HD, 2>();
  if (e == cudaSuccess) e = configure_one<__nv_bfloat16, HD, 4>();
  return e;
}

// Cuts the blocks of bn slots of all (sequence, KV head, tile of rt rows) into at most as
// many CTAs as SMs, runs `main` over them, and joins the splits.
template <int HD, typename Main>
cudaError_t launch_split(const TreeAttnArgs& a, const TreeAttnShape& s, int rt, int bn, int sms, int* launches,
                         cudaStream_t st, Main main) {
  TAKernelArgs P;
  P.a = a;
  const int G = a.nq / a.kvh;
  auto tiles = [&](int m) { return (m * G + rt - 1) / rt; };
  auto blocks = [&](int i) { return s.seqs[i].m ? (s.t0[i] + s.seqs[i].m + bn - 1) / bn : 0; };
  long long total = 0, items = 0;
  for (int i = 0; i < a.n_seqs; ++i) {
    const long long per = (long long)a.kvh * tiles(s.seqs[i].m);
    total += blocks(i) * per;
    items += per;
  }
  // blocks per split: the fewest with which all CTAs run at once (short last splits make
  // that a little more than total / sms); with more items than SMs, about one SM's share
  P.bps = (int)std::max<long long>(1, (total + sms - 1) / sms);
  for (int step = 0; items < sms && step < 256; ++step) {
    long long ctas = 0;
    for (int i = 0; i < a.n_seqs; ++i) ctas += (blocks(i) + P.bps - 1) / P.bps * (long long)a.kvh * tiles(s.seqs[i].m);
    if (ctas <= sms) break;
    P.bps += 1 + P.bps / 64;
  }
  int splits = 1;
  size_t part = 0;
  for (int i = 0; i < a.n_seqs; ++i) {
    P.seq[i] = s.seqs[i].seq;
    P.row0[i] = s.seqs[i].row0;
    P.m[i] = s.seqs[i].m;
    P.t0[i] = s.t0[i];
    const int m = s.seqs[i].m, ns = m ? ta_splits(s.t0[i] + m, bn, P.bps) : 1;
    P.part0[i] = (int)part;
    if (ns > 1) part += (size_t)ns * m * a.nq;
    splits = std::max(splits, ns);
  }
  cudaError_t e = main(P, dim3(splits, a.kvh * tiles(s.max_m), a.n_seqs));
  *launches += 1;
  if (e != cudaSuccess || splits == 1) return e;
  const int rows = s.max_m * a.nq;  // rows and query heads of a sequence
  const bool many = splits > 8;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(many ? rows : (rows + 7) / 8, a.n_seqs);
  cfg.blockDim = dim3(256);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  *launches += 1;
  return cudaLaunchKernelEx(&cfg, many ? tree_join_kernel<HD, 8> : tree_join_kernel<HD, 1>, P, bn);
}

template <typename KT, int HD, int WR>
cudaError_t launch(const TreeAttnArgs& a, const TreeAttnShape& s, int sms, int* launches, cudaStream_t st) {
  using T = MmaTile<KT, HD, WR>;
  return launch_split<HD>(a, s, T::RT, T::BN, sms, launches, st, [&](const TAKernelArgs& P, dim3 grid) {
    tree_attn_kernel<KT, HD, WR><<<grid, kTAThreads, T::kSmem, st>>>(P);
    return cudaGetLastError();
  });
}

// Few rows take the mma.sync tiles of 16 and 32 rows: their CTAs start faster, and up to
// there they keep up with HBM (28 query heads on 4 KV heads of 128, us with mma.sync /
// tcgen05: 3 nodes at 2000 slots 12.6 / 16.7, at 16000 20.7 / 24.1). Tiles of 64 rows pay on
// a bf16 cache while no SM has more than two blocks (9 nodes at 2000 slots 14.5 / 18.6, 16
// nodes there 16.9 / 20.7, at 3500 22.5 / 18.7; 32 nodes at 300 slots 14.7 / 18.6; on an
// fp32 cache 8 nodes at 2000 slots 18.6 / 16.6). The rest runs on tcgen05.
template <typename KT, int HD>
cudaError_t launch_hd(const TreeAttnArgs& a, const TreeAttnShape& s, int sms, int* launches, cudaStream_t st) {
  const int rows = s.max_m * (a.nq / a.kvh);  // rows of the largest sequence that share a KV head
  if (rows <= 16) return launch<KT, HD, 1>(a, s, sms, launches, st);
  if (rows <= 32) return launch<KT, HD, 2>(a, s, sms, launches, st);
  if constexpr (sizeof(KT) == 2) {
    long long blocks = 0;
    for (int i = 0; i < a.n_seqs; ++i)
      if (s.seqs[i].m) blocks += (long long)((s.t0[i] + s.seqs[i].m + kTcBlock - 1) / kTcBlock) * a.kvh;
    if ((rows + 63) / 64 * blocks <= 2ll * sms) return launch<KT, HD, 4>(a, s, sms, launches, st);
  }
  return launch_split<HD>(a, s, kTcRows, kTcBlock, sms, launches, st, [&](const TAKernelArgs& P, dim3 grid) {
    return sizeof(KT) == 2 ? launch_tree_attn_tc(P, HD, grid, st) : launch_tree_attn_tc32(P, HD, grid, st);
  });
}

}  // namespace

// With bps >= total / sms a sequence of more than one split has at most 2 blocks / bps of
// them, so the split sequences' CTAs are at most 2 sms, each with up to 128 rows.
size_t tree_attn_part_rows(int sms) { return (size_t)2 * sms * 128; }

cudaError_t configure_tree_attn() {
  cudaError_t e = configure_hd<64>();
  if (e == cudaSuccess) e = configure_hd<128>();
  if (e == cudaSuccess) e = configure_tree_attn_tc();
  if (e == cudaSuccess) e = configure_tree_attn_tc32();
  return e;
}

cudaError_t op_tree_attention(const TreeAttnArgs& a, const TreeAttnShape& s, int kv_dtype, int hd, int sms,
                              int* launches, cudaStream_t st) {
  // what the kernels use without asking; err only after a wait that gave up
  if (!a.tc_k || !a.tc_v || !a.part_o || !a.part_ml || !a.err) return cudaErrorInvalidValue;
  if (kv_dtype == 0) return hd == 64 ? launch_hd<float, 64>(a, s, sms, launches, st)
                                     : launch_hd<float, 128>(a, s, sms, launches, st);
  return hd == 64 ? launch_hd<__nv_bfloat16, 64>(a, s, sms, launches, st)
                  : launch_hd<__nv_bfloat16, 128>(a, s, sms, launches, st);
}

}  // namespace dllm
