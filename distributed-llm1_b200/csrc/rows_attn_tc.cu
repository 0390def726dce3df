// rows_attn_tc.cu — attention of a batch's long chunks over a paged cache, on tcgen05.
//
// The mathematics are rows_attn.cu's. Two kernels:
//
// rows_planes_kernel brings the K and V rows that a sequence's rows see into fp16 once, before
// the many tiles that read them: per (KV head, block of slots) one power of two takes the
// largest value below 2^15, and a value becomes one fp16 (bf16 caches: 8 significant bits fit)
// or two (fp32 and 4-bit caches: 22 bits). What falls below fp16's range is 2^-32 of the
// block's largest value at most. A block is written as the image that shared memory needs:
// 128 rows (128 slots, or 64 slots and their second terms) in swizzled boxes of 64 dims, so
// the main kernel fetches it with one bulk copy and knows no page table.
//
// rows_tc_kernel: one CTA per 256 rows (query head and token) that share a KV head, two
// tiles of 128, over all their blocks or a share of them:
//   producer (1 warp)   bulk copies of K(0), V(0), K(1), V(1) ... into a ring
//   MMA (1 warp)        S = q K^T per tile and block, O = P V
//   two softmax groups  128 threads each, one row per thread: S from tensor memory, online
//                       softmax, P back over S as two fp16 terms, then O into registers
// q and p run as two fp16 terms too (22 bits; each row of q by its own power of two, p as
// 2^15 p), so a product takes two MMAs where K and V are one plane, three where they are two:
// the low terms first, so that only the last ones add at full size (the tensor core
// truncates each addition); a block's P V starts from zero and the blocks are added in fp32
// registers. With two planes S takes q_high (K_high | K_low) as one MMA of N = 128, and
// q_low K_high goes to the K_low half; the softmax adds the halves.
// Tensor memory: S and P of both tiles 2 x 128 columns, O 2 x 128.
#include <algorithm>

#include "rows_attn_tc.cuh"
#include "tc.cuh"

namespace dllm {
namespace {

// ---- K and V as fp16 planes ------------------------------------------------------------------
constexpr int kPlaneThreads = 256;

// Eight values of one row, from 8 dims on.
template <int KIND, int HD>
DLLM_DEV void load8(const void* rows, const uint32_t* pairs, size_t row, int c, float (&x)[8]) {
  if constexpr (KIND == kKvF32) {
    const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(rows) + row * HD + c * 8);
    const float4 a = p[0], b = p[1];
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
  } else if constexpr (KIND == kKvBf16) {
    const uint4 a = reinterpret_cast<const uint4*>(rows)[row * (HD / 8) + c];
    x[0] = bf16_lo(a.x), x[1] = bf16_hi(a.x), x[2] = bf16_lo(a.y), x[3] = bf16_hi(a.y);
    x[4] = bf16_lo(a.z), x[5] = bf16_hi(a.z), x[6] = bf16_lo(a.w), x[7] = bf16_hi(a.w);
  } else {
    const uint32_t w = static_cast<const uint32_t*>(rows)[row * (HD / 8) + c], pr = pairs[row * (HD / kGroup4) + c / 4];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = fmaf((float)(w >> (4 * e) & 15u), bf16_lo(pr), bf16_hi(pr));
  }
}

// Grid: (KV head, block, K or V) of every sequence in turn.
template <int KIND, int HD>
__global__ void __launch_bounds__(kPlaneThreads) rows_planes_kernel(const __grid_constant__ RowsKernelArgs P) {
  using T = TcTile<KIND, HD>;
  constexpr int C = HD / 8, kEach = T::BN * C / kPlaneThreads;
  __shared__ float smax[kPlaneThreads / 32];
  __shared__ int sbad;
  const RowsAttnArgs& a = P.a;
  const int which = blockIdx.x & 1, at = blockIdx.x >> 1, i = rows_find(P.unit0, P.n_seqs, at);
  const RowsView v(P.t0[i], P.t0[i] + P.m[i] - 1, a.window, a.sinks, T::BN);
  const int head = (at - P.unit0[i]) / v.nb, s0 = v.slot0((at - P.unit0[i]) % v.nb, T::BN), end = v.p1 + 1;
  const int tid = threadIdx.x;
  const void* rows = which ? a.vc : a.kc;
  const uint32_t* pairs = which ? a.vs : a.ks;
  if (tid == 0) sbad = 0;
  float x[kEach][8], m = 0.f;
  bool bad = false;
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    const int j = tid + e * kPlaneThreads, slot = s0 + j / C;
#pragma unroll
    for (int u = 0; u < 8; ++u) x[e][u] = 0.f;
    if (slot < end) load8<KIND, HD>(rows, pairs, a.pages.row(P.seq[i], slot, head), j % C, x[e]);
  }
#pragma unroll
  for (int e = 0; e < kEach; ++e)
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const bool fine = is_finite(x[e][u]);
      m = fmaxf(m, fine ? fabsf(x[e][u]) : 0.f);
      bad |= !fine;
      // 0 x NaN would reach rows that do not see the slot; the main kernel adds such values of V
      // to the rows that do
      if (which && !fine) x[e][u] = 0.f;
    }
  m = warp_max(m);
  if (tid % 32 == 0) smax[tid / 32] = m;
  __syncthreads();
  if (bad) sbad = 1;
#pragma unroll
  for (int w = 0; w < kPlaneThreads / 32; ++w) m = fmaxf(m, smax[w]);
  // in steps of 2^8, so that neighbouring blocks hardly ever differ
  const int ex = max((int)(__float_as_uint(m) >> 23) | 7, 15);
  const float up = power_of_two(268 - ex);
  unsigned char* image = static_cast<unsigned char*>(a.planes) + (size_t)blockIdx.x * T::kTile;
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    const int j = tid + e * kPlaneThreads, row = j / C, c = j % C;
    uint32_t h[4], l[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) split2_f16(x[e][2 * u] * up, x[e][2 * u + 1] * up, h[u], l[u]);
    unsigned char* p = image + (c / 8) * T::kBox + row * 128 + (((c & 7) ^ (row & 7)) << 4);
    *reinterpret_cast<uint4*>(p) = make_uint4(h[0], h[1], h[2], h[3]);
    if constexpr (T::kPlanes == 2) *reinterpret_cast<uint4*>(p + T::BN * 128) = make_uint4(l[0], l[1], l[2], l[3]);
  }
  __syncthreads();
  if (tid == 0) {
    float2* info = static_cast<float2*>(a.info) + blockIdx.x;
    *info = make_float2(power_of_two(ex - 14), sbad ? 1.f : 0.f);
  }
}

// ---- the main kernel ---------------------------------------------------------------------------
struct TcShared {
  uint64_t full[kTcRing], empty[kTcRing];
  uint64_t s_full[2], p_ready[2], o_full[2];
  uint64_t idle;
  uint32_t tmem;
  volatile int abort;
  float back[kTcTileRows];  // what a row of q was divided by, times 2^14
};

// 32 columns of this thread's lane to tensor memory.
DLLM_DEV void tmem_st32(uint32_t addr, const uint32_t (&h)[16], const uint32_t (&l)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
      "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};" ::"r"(h[0]),
      "r"(h[1]), "r"(h[2]), "r"(h[3]), "r"(h[4]), "r"(h[5]), "r"(h[6]), "r"(h[7]), "r"(h[8]), "r"(h[9]), "r"(h[10]),
      "r"(h[11]), "r"(h[12]), "r"(h[13]), "r"(h[14]), "r"(h[15]), "r"(l[0]), "r"(l[1]), "r"(l[2]), "r"(l[3]), "r"(l[4]),
      "r"(l[5]), "r"(l[6]), "r"(l[7]), "r"(l[8]), "r"(l[9]), "r"(l[10]), "r"(l[11]), "r"(l[12]), "r"(l[13]), "r"(l[14]),
      "r"(l[15]), "r"(addr)
      : "memory");
}
DLLM_DEV void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

template <int KIND, int HD>
__global__ void __launch_bounds__(kTcThreads, 1) rows_tc_kernel(const __grid_constant__ RowsKernelArgs P) {
  using T = TcTile<KIND, HD>;
  constexpr int BN = T::BN, BOX = T::BOX;
  extern __shared__ unsigned char smem_raw[];
  __shared__ __align__(8) TcShared sh;
  const RowsAttnArgs& a = P.a;
  asm volatile("griddepcontrol.launch_dependents;");  // the join may be scheduled; it waits for this grid's end
  const RowsTile k(P, blockIdx.x, kTcTileRows, BN);
  if (k.split >= k.nsplit) return;
  const int nb = k.b1 - k.b0;
  const int tiles = k.R - k.r0 > 128 ? 2 : 1;

  // the warp's number as a value that is the same in all its lanes by construction
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  unsigned char* base = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  unsigned char* sQ = base;  // [tile][term][box][128 rows][128 bytes]
  unsigned char* ring = base + 4 * T::kTile;

  // number of a block among the sequence's (KV head, block) pairs
  const RowsView all(k.t0, k.t0 + k.m - 1, a.window, a.sinks, BN);
  const int unit0 = P.unit0[k.i] + k.head * all.nb;
  auto unit_of = [&](int s0) {
    const int blk = s0 / BN;
    return unit0 + (blk >= all.first ? blk - all.first + all.nsink : blk);
  };

  if (tid == 0) {
    for (int s = 0; s < T::kRing; ++s) mbar_init(&sh.full[s], 1), mbar_init(&sh.empty[s], 1);
    for (int w = 0; w < 2; ++w) mbar_init(&sh.s_full[w], 1), mbar_init(&sh.p_ready[w], 128), mbar_init(&sh.o_full[w], 1);
    mbar_init(&sh.idle, 1);
    sh.abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 8) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem)), "r"(512u));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, sh.tmem, 0);

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    if (warp == 8 && lane == 0) {
      // ---- producer: tile t is K of block t / 2 (even) or V
      int sent = 0;
      const unsigned char* planes = static_cast<const unsigned char*>(a.planes);
      for (int t = 0; t < 2 * nb; ++t) {
        const int s = t % T::kRing;
        if (!wait_phase(&sh.empty[s], ((uint32_t)(t / T::kRing) & 1u) ^ 1u, &sh.abort)) break;  // nothing is loaded over memory that may still be read
        mbar_expect_tx(&sh.full[s], T::kTile);
        bulk_load(ring + s * T::kTile, planes + ((size_t)unit_of(k.v.slot0(k.b0 + t / 2, BN)) * 2 + (t & 1)) * T::kTile, T::kTile,
                  &sh.full[s]);
        sent = t + 1;
      }
      // whatever happened to the others, the copies under way land before the CTA ends
      for (int t = max(0, sent - T::kRing); t < sent; ++t) mbar_wait(&sh.full[t % T::kRing], (uint32_t)(t / T::kRing) & 1u);
    } else if (warp == 9) {
      // ---- MMA issuer. The whole warp runs the loop and one elected lane issues, so that the
      // operands stay in uniform registers.
      asm volatile("bar.sync 2, 288;" ::: "memory");  // q is there
      const uint32_t leader = elect_one();
      const uint32_t idesc = (1u << 4) | ((uint32_t)(128 >> 4) << 24);                // fp32 += fp16 x fp16, M = 128
      const uint32_t id_s = idesc | ((uint32_t)(128 >> 3) << 17);                     // N = 128 rows of K, K-major
      const uint32_t id_half = idesc | ((uint32_t)(64 >> 3) << 17);                   // the first 64 of them
      const uint32_t id_o = idesc | ((uint32_t)(HD >> 3) << 17) | (1u << 16);         // N = dims, B with N contiguous
      auto full = [&](int t) {
        wait_phase(&sh.full[t % T::kRing], (uint32_t)(t / T::kRing) & 1u, &sh.abort);
        tc_fence_after();
      };
      auto scores = [&](int w, int n) {
        if (leader) {
          const unsigned char* kb = ring + (2 * n % T::kRing) * T::kTile;
          const unsigned char* qb = sQ + w * 2 * T::kTile;
          const uint32_t d = tmem + (uint32_t)w * 128;
          // the low term of q first; with two planes of K it comes second, into their half
#pragma unroll
          for (int term = 0; term < 2; ++term)
#pragma unroll
            for (int x = 0; x < BOX; ++x)
#pragma unroll
              for (int kk = 0; kk < 4; ++kk) {
                const uint64_t bd = umma_desc_sw128(kb + x * T::kBox) + 2ull * kk;
                const int plane = T::kPlanes == 1 ? 1 - term : term;
                const uint64_t ad = umma_desc_sw128(qb + plane * T::kTile + x * T::kBox) + 2ull * kk;
                if (T::kPlanes == 2 && term == 1) umma_bf16(d + 64, ad, bd, id_half, 1u);
                else umma_bf16(d, ad, bd, id_s, (uint32_t)(term || x || kk));
              }
          if (w == tiles - 1) umma_commit(&sh.empty[2 * n % T::kRing]);
          umma_commit(&sh.s_full[w]);
        }
        __syncwarp();
      };
      full(0);
      for (int w = 0; w < tiles; ++w) scores(w, 0);
      for (int n = 0; n < nb; ++n) {
        for (int w = 0; w < tiles; ++w) {
          if (w == 0) full(2 * n + 1);
          wait_phase(&sh.p_ready[w], (uint32_t)n & 1u, &sh.abort);  // (P is there, and O of the block before has been read)
          tc_fence_after();
          if (leader) {
            const int s = (2 * n + 1) % T::kRing;
            const unsigned char* vb = ring + s * T::kTile;
            const uint32_t p = tmem + (uint32_t)w * 128, d = tmem + 256u + (uint32_t)w * 128;
            // products (term of p, plane of V), the smallest first
#pragma unroll
            for (int i = 0; i < T::kPlanes + 1; ++i) {
              const int low = i == 0, plane = T::kPlanes == 2 && i == 1;
              const uint64_t bd = umma_desc_mn_sw128(vb + plane * (BN * 128), T::kBox);
#pragma unroll
              for (int ks = 0; ks < BN / 16; ++ks)  // 16 slots: 2048 bytes on
                umma_bf16_ts(d, p + 32u * (ks / 2) + 8u * (ks % 2) + 16u * low, bd + 128ull * ks, id_o, (uint32_t)(i || ks));
            }
            if (w == tiles - 1) umma_commit(&sh.empty[s]);
            umma_commit(&sh.o_full[w]);
          }
          __syncwarp();
          if (n + 1 < nb) {
            if (w == 0) full(2 * n + 2);
            // the next scores replace P
            wait_phase(&sh.o_full[w], (uint32_t)n & 1u, &sh.abort);
            tc_fence_after();
            scores(w, n + 1);
          }
        }
      }
      // nothing of this warp's is under way when the tensor memory is freed
      if (leader) umma_commit(&sh.idle);
      __syncwarp();
      mbar_wait(&sh.idle, 0u);
    }
    __syncwarp();
  } else {
    // ---- q: rows scaled so that the softmax is in powers of two, each divided by a power of two
    // next to its largest element, as two fp16 terms. Rows behind the last one are zero.
    asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    {
      constexpr int C = HD / 8, kPass = 256 / C, kBatch = 4;  // C threads per row
      const int c = tid % C;
#pragma unroll 1
      for (int r1 = tid / C; r1 < kTcTileRows; r1 += kPass * kBatch) {
        float x[kBatch][8];
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
          const int r = k.r0 + r1 + u * kPass;
#pragma unroll
          for (int e = 0; e < 8; ++e) x[u][e] = 0.f;
          if (r < k.R) load8<kKvF32, HD>(a.q, nullptr, (size_t)k.row0 * a.nq + k.place(r, a.nq), c, x[u]);
        }
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
          const int row = r1 + u * kPass;
          float m = 0.f;
#pragma unroll
          for (int e = 0; e < 8; ++e) x[u][e] *= a.scale_log2, m = fmaxf(m, fabsf(x[u][e]));
#pragma unroll
          for (int d = C / 2; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
          const int ex = min(max((int)(__float_as_uint(m) >> 23), 15), 254);
          const float up = power_of_two(268 - ex);
          uint32_t h[4], l[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) split2_f16(x[u][2 * e] * up, x[u][2 * e + 1] * up, h[e], l[e]);
          unsigned char* p = sQ + (row / 128) * 2 * T::kTile + (c / 8) * T::kBox + (row % 128) * 128 + (((c & 7) ^ (row & 7)) << 4);
          *reinterpret_cast<uint4*>(p) = make_uint4(h[0], h[1], h[2], h[3]);
          *reinterpret_cast<uint4*>(p + T::kTile) = make_uint4(l[0], l[1], l[2], l[3]);
          if (c == 0) sh.back[row] = power_of_two(ex - 14);
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // q is read by the MMA
      asm volatile("bar.sync 2, 288;" ::: "memory");
    }
    // ---- softmax: group w, one row per thread
    const int w = warp >> 2, r = k.r0 + tid, slot = k.slot_of(r);
    const uint32_t lanes = tmem + (uint32_t)w * 128 + ((uint32_t)((warp & 3) * 32) << 16);
    float o[HD], m = -INFINITY, l = 0.f, unit = 0.f;
#pragma unroll
    for (int d = 0; d < HD; ++d) o[d] = 0.f;
    if (w < tiles) {
      const float back = sh.back[tid];
      // the rows of this tile see slots up to p0 at least, and from p1 - window on
      const int p0 = k.t0 + (k.r0 + w * 128) / k.G, p1 = k.t0 + (min(k.r0 + w * 128 + 128, k.R) - 1) / k.G;
      const float2* info = static_cast<const float2*>(a.info);
      int s0 = k.v.slot0(k.b0, BN);
      float4 next = __ldg(reinterpret_cast<const float4*>(info + 2 * (size_t)unit_of(s0)));
      for (int n = 0; n < nb; ++n) {
        const float4 now = next;  // factor of K, -, factor of V, whether V had other than numbers
        const int s_now = s0;
        if (n + 1 < nb) {
          s0 = k.v.slot0(k.b0 + n + 1, BN);
          next = __ldg(reinterpret_cast<const float4*>(info + 2 * (size_t)unit_of(s0)));
        }
        const float f = back * now.x;
        const bool edge = s_now + BN - 1 > p0 || (s_now <= p1 - a.window && s_now + BN > a.sinks);
        // column c is visible where c <= last and (c >= first or c < sink)
        const int last = slot - s_now, first = last >= a.window ? last - a.window + 1 : 0, sink = a.sinks - s_now;
        wait_phase(&sh.s_full[w], (uint32_t)n & 1u, &sh.abort);
        tc_fence_after();
        // 32 scores from column c on, hidden ones at -inf
        auto load = [&](int c, uint32_t(&u)[32]) {
          tmem_ld32(lanes + (uint32_t)c, u);
          if constexpr (T::kPlanes == 2) {
            uint32_t z[32];
            tmem_ld32(lanes + 64u + (uint32_t)c, z);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 32; ++e) u[e] = __float_as_uint(__uint_as_float(u[e]) + __uint_as_float(z[e]));
          } else {
            tmem_ld_wait();
          }
          if (edge) {
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (!(c + e <= last && (c + e >= first || c + e < sink))) u[e] = 0xff800000u;
          }
        };
        float x0 = -INFINITY, x1 = -INFINITY, x2 = -INFINITY, x3 = -INFINITY;
#pragma unroll
        for (int c = 0; c < BN; c += 32) {
          uint32_t u[32];
          load(c, u);
#pragma unroll
          for (int e = 0; e < 32; e += 4) {
            x0 = fmaxf(x0, __uint_as_float(u[e])), x1 = fmaxf(x1, __uint_as_float(u[e + 1]));
            x2 = fmaxf(x2, __uint_as_float(u[e + 2])), x3 = fmaxf(x3, __uint_as_float(u[e + 3]));
          }
        }
        const float x = fmaxf(m, fmaxf(fmaxf(x0, x1), fmaxf(x2, x3)) * f);
        const float b = x == -INFINITY ? 0.f : x;  // a row that has seen nothing: every p is 0
        float g = ex2(m - b);
        const float shift = 15.f - b;
        m = x;
        float sum0 = 0.f, sum1 = 0.f;
#pragma unroll
        for (int c = 0; c < BN; c += 32) {
          uint32_t u[32], ph[16], pl[16];
          load(c, u);
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const float q0 = ex2(fmaf(__uint_as_float(u[2 * e]), f, shift)), q1 = ex2(fmaf(__uint_as_float(u[2 * e + 1]), f, shift));
            sum0 += q0, sum1 += q1;
            split2_f16(q0, q1, ph[e], pl[e]);
          }
          tmem_st32(lanes + (uint32_t)c, ph, pl);
        }
        l = fmaf(l, g, sum0 + sum1);
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(&sh.p_ready[w]);
        // o is in units of `unit`, a power of two that only grows
        float drop = 1.f;
        if (now.z != unit) {
          const float to = fmaxf(now.z, unit);
          g *= unit / to, drop = now.z / to, unit = to;
        }
        wait_phase(&sh.o_full[w], (uint32_t)n & 1u, &sh.abort);
        tc_fence_after();
#pragma unroll
        for (int d = 0; d < HD; d += 32) {
          uint32_t u[32];
          tmem_ld32(lanes + 256u + (uint32_t)d, u);
          tmem_ld_wait();
          if (drop != 1.f) {
#pragma unroll
            for (int e = 0; e < 32; ++e) u[e] = __float_as_uint(__uint_as_float(u[e]) * drop);
          }
#pragma unroll
          for (int e = 0; e < 32; ++e) o[d + e] = fmaf(o[d + e], g, __uint_as_float(u[e]));
        }
        tc_fence_before();
        if (now.w != 0.f) {
#pragma unroll 1
          for (int c = 0; c < BN; ++c) {
            if (!(c <= last && (c >= first || c < sink))) continue;
            const size_t row = a.pages.row(k.seq, s_now + c, k.head);
#pragma unroll
            for (int d = 0; d < HD; d += 8) {
              float v[8];
              load8<KIND, HD>(a.vc, a.vs, row, d / 8, v);
#pragma unroll
              for (int e = 0; e < 8; ++e)
                if (!is_finite(v[e])) o[d + e] += v[e];
            }
          }
        }
      }
    }
    // every MMA has completed (each group waited for its last O): the operands' memory is free
    asm volatile("bar.sync 1, 256;" ::: "memory");
    float* sO = reinterpret_cast<float*>(base);
    float* sML = sO + kTcTileRows * (HD + 4);
    float* mine = sO + tid * (HD + 4);
#pragma unroll
    for (int d = 0; d < HD; d += 4)
      *reinterpret_cast<float4*>(mine + d) = make_float4(o[d] * unit, o[d + 1] * unit, o[d + 2] * unit, o[d + 3] * unit);
    sML[tid * 2] = m, sML[tid * 2 + 1] = l;
    asm volatile("bar.sync 1, 256;" ::: "memory");
    if (!sh.abort) rows_finish<HD, 1, kTcTileRows, 256>(P, k, sO, sML, tid);
  }
  tc_fence_before();
  __syncthreads();
  if (tid == 0 && sh.abort) atomicExch(a.err, kErrRowsWait);
  if (warp == 8) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u));
  }
}

template <int KIND, int HD>
cudaError_t launch(const RowsKernelArgs& P, int ctas, int units, cudaStream_t st) {
  rows_planes_kernel<KIND, HD><<<2 * units, kPlaneThreads, 0, st>>>(P);
  rows_tc_kernel<KIND, HD><<<ctas, kTcThreads, TcTile<KIND, HD>::kSmem, st>>>(P);
  return cudaGetLastError();
}

template <int KIND, int HD>
cudaError_t configure() {
  return cudaFuncSetAttribute(rows_tc_kernel<KIND, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, TcTile<KIND, HD>::kSmem);
}

}  // namespace

cudaError_t configure_rows_attn_tc() {
  cudaError_t e = configure<kKvF32, 64>();
  if (e == cudaSuccess) e = configure<kKvF32, 128>();
  if (e == cudaSuccess) e = configure<kKvBf16, 64>();
  if (e == cudaSuccess) e = configure<kKvBf16, 128>();
  if (e == cudaSuccess) e = configure<kKv4, 64>();
  if (e == cudaSuccess) e = configure<kKv4, 128>();
  return e;
}

cudaError_t launch_rows_tc(const RowsKernelArgs& P, int kind, int hd, int ctas, int units, cudaStream_t st) {
  switch (kind) {
    case kKvF32: return hd == 64 ? launch<kKvF32, 64>(P, ctas, units, st) : launch<kKvF32, 128>(P, ctas, units, st);
    case kKvBf16: return hd == 64 ? launch<kKvBf16, 64>(P, ctas, units, st) : launch<kKvBf16, 128>(P, ctas, units, st);
    default: return hd == 64 ? launch<kKv4, 64>(P, ctas, units, st) : launch<kKv4, 128>(P, ctas, units, st);
  }
}

}  // namespace dllm
