// rows_attn_tc.cu — attention of a batch's long chunks over a paged cache, on tcgen05.
//
// The mathematics are rows_attn.cu's. Two kernels:
//
// rows_planes_kernel brings the K and V rows that a sequence's rows see into fp16 once, before
// the many tiles that read them: per (KV head, block of slots) one power of two takes the
// largest value below 2^15, and a value becomes one fp16 (bf16 caches: 8 significant bits fit)
// or two (fp32 and 4-bit caches), which keep 22 bits of the largest value of every slot. Where
// some slot of a block lies too far below another for that ("wide" blocks), each slot has a power of
// two of its own: a large value in a slot that a row does not see takes no bits from those that it sees.
// The softmax then multiplies the scores by K's powers, and brings V's into p, relative to the largest
// of the slots that the row sees. A block is written as the image that shared memory needs:
// 128 rows (128 slots, or 64 slots and their second terms) in swizzled boxes of 64 dims, so
// the main kernel fetches it with one bulk copy and knows no page table.
//
// rows_tc_kernel: one CTA per SM takes an equal share of all blocks, a segment after the other:
// 256 rows (query head and token) that share a KV head, two tiles of 128, over all their blocks
// or some. (A CTA per 256 rows left a quarter of the SMs idle with 224 of them.)
//   producer (1 warp)   bulk copies of K(0), V(0), K(1), V(1) ... into a ring, across segments
//   MMA (1 warp)        S = q K^T per tile and block, O = P V
//   two softmax groups  128 threads each, one row per thread: S from tensor memory, online
//                       softmax, P back over S as two fp16 terms, then O into registers
// q and p run as two fp16 terms too (22 bits; each row of q by its own power of two, p between
// 2^8 and 2^15 at its largest), so a product takes two MMAs where K and V are one plane, three where they are two:
// the low terms first, so that only the last ones add at full size (the tensor core
// truncates each addition); a block's P V starts from zero and the blocks are added in fp32
// registers. With two planes S takes q_high (K_high | K_low) as one MMA of N = 128, and
// q_low K_high goes to the K_low half; the softmax adds the halves.
// Tensor memory: S and P of both tiles 2 x 128 columns, O 2 x 128.
// What bounds it: the products and, between them, the softmax. A chunk of 2048 rows of 28 heads of 128
// under a 4096-token window, bf16: 220 us in the main kernel, 546 TFLOP/s of the floor's one product
// per operand, tensor pipe 66 % busy; over 8148 4-bit slots 484 us, 432 TFLOP/s, 70 %. (The code of wide
// blocks, which no block of these needs, takes 2 % of the first by its mere presence. With every block wide the
// two take 561 and 1004 us with their launches instead of 224 and 461.)
// The main kernel starts while the planes are written (its CTAs set up and bring q), and waits for
// that grid's end before it reads them (a prompt of 1501 rows: 47 -> 43 us with its launches).
#include "rows_attn_tc.cuh"
#include "tc.cuh"

namespace dllm {
namespace {

// ---- K and V as fp16 planes ------------------------------------------------------------------
constexpr int kPlaneEach = 2;  // units of 8 dims per thread (8 and 256 threads per block: 15 us for 400 blocks, 10 so; 11 with the slots' maxima)
template <int KIND, int HD>
constexpr int kPlaneThreads = TcTile<KIND, HD>::BN * (HD / 8) / kPlaneEach;

// What the main kernel is told of a block's K or V, 16 bits: the exponent of its power of two, whether it
// had values that are no numbers, whether it has powers per slot.
constexpr uint32_t kTcBad = 1u << 8, kTcWide = 1u << 9;

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
__global__ void __launch_bounds__(kPlaneThreads<KIND, HD>, 2048 / kPlaneThreads<KIND, HD>) rows_planes_kernel(const __grid_constant__ RowsKernelArgs P) {
  using T = TcTile<KIND, HD>;
  constexpr int C = HD / 8, kEach = kPlaneEach, kThreads = kPlaneThreads<KIND, HD>;
  __shared__ uint32_t smost[kThreads / 32], sleast[kThreads / 32];
  __shared__ int sbad;
  const RowsAttnArgs& a = P.a;
  asm volatile("griddepcontrol.launch_dependents;");  // the main kernel may start; it waits for this grid's end
  const int which = blockIdx.x & 1, at = blockIdx.x >> 1, i = rows_find(P.unit0, P.n_seqs, at);
  const RowsView v(P.t0[i], P.t0[i] + P.m[i] - 1, a.window, a.sinks, T::BN);
  const int head = (at - P.unit0[i]) / v.nb, s0 = v.slot0((at - P.unit0[i]) % v.nb, T::BN), end = v.p1 + 1;
  const int tid = threadIdx.x;
  const void* rows = which ? a.vc : a.kc;
  const uint32_t* pairs = which ? a.vs : a.ks;
  if (tid == 0) sbad = 0;
  float x[kEach][8];
  uint32_t m[kEach];
  bool bad = false;
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    const int j = tid + e * kThreads, slot = s0 + j / C;
#pragma unroll
    for (int u = 0; u < 8; ++u) x[e][u] = 0.f;
    if (slot < end) load8<KIND, HD>(rows, pairs, a.pages.row(P.seq[i], slot, head), j % C, x[e]);
  }
  // the largest magnitude of each slot (C lanes side by side), and of the block's slots the most and
  // the least that is not zero: positive numbers in the order of their bits
  uint32_t most = 0u, least = ~0u;
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    m[e] = 0u;
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const bool fine = is_finite(x[e][u]);
      m[e] = max(m[e], fine ? __float_as_uint(fabsf(x[e][u])) : 0u);
      bad |= !fine;
      // 0 x NaN would reach rows that do not see the slot; the main kernel adds such values of V
      // to the rows that do
      if (which && !fine) x[e][u] = 0.f;
    }
#pragma unroll
    for (int d = C / 2; d > 0; d >>= 1) m[e] = max(m[e], __shfl_xor_sync(0xffffffffu, m[e], d));
    most = max(most, m[e]), least = min(least, m[e] ? m[e] : ~0u);
  }
  most = __reduce_max_sync(0xffffffffu, most), least = __reduce_min_sync(0xffffffffu, least);
  if (tid % 32 == 0) smost[tid / 32] = most, sleast[tid / 32] = least;
  __syncthreads();
  if (bad) sbad = 1;
  const bool has = tid % 32 < kThreads / 32;
  most = __reduce_max_sync(0xffffffffu, has ? smost[tid % 32] : 0u);
  least = __reduce_min_sync(0xffffffffu, has ? sleast[tid % 32] : ~0u);
  // The block's power of two goes in steps of 2^8, so that neighbouring blocks hardly ever differ. With it,
  // the largest value of a slot lies above 2^-3 if its exponent is ex - 17 or more, and what two fp16 terms
  // lose, 2^-25, is 2^-22 of it.
  const int ex = max((int)(most >> 23) | 7, 15);
  const bool wide = (int)(least >> 23) < ex - 17;
  unsigned char* image = static_cast<unsigned char*>(a.planes) + (size_t)blockIdx.x * T::kTile;
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    const int j = tid + e * kThreads, row = j / C, c = j % C;
    const int own = wide ? max((int)(m[e] >> 23), 15) : ex;
    const float up = power_of_two(268 - own);
    uint32_t h[4], l[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) split2_f16(x[e][2 * u] * up, x[e][2 * u + 1] * up, h[u], l[u]);
    unsigned char* p = image + (c / 8) * T::kBox + row * 128 + (((c & 7) ^ (row & 7)) << 4);
    *reinterpret_cast<uint4*>(p) = make_uint4(h[0], h[1], h[2], h[3]);
    if constexpr (T::kPlanes == 2) *reinterpret_cast<uint4*>(p + T::BN * 128) = make_uint4(l[0], l[1], l[2], l[3]);
    if (wide && c == 0) a.exps[(size_t)blockIdx.x * kTcExps + row] = (unsigned char)own;
  }
  __syncthreads();
  if (tid == 0) a.info[blockIdx.x] = (uint16_t)((uint32_t)ex | (sbad ? kTcBad : 0u) | (wide ? kTcWide : 0u));
}

// ---- the main kernel ---------------------------------------------------------------------------
struct TcShared {
  uint64_t empty[kTcRing];
  // What the MMA warp waits for, one barrier at a time: the first tile's P and V, its O and the next
  // K (both in turn, so that the producer may run ahead), the second tile's P, its O.
  uint64_t pv_ready[kTcTurns], ok_ready[kTcTurns], p1_ready, o1_done;
  uint64_t q_ready[2];
  uint64_t s_full[2], o_full[2];  // the softmax groups' side
  uint64_t idle;
  uint32_t tmem;
  volatile int abort;
  float back[kTcTileRows];  // what a row of q was divided by, times 2^14
};
static_assert(sizeof(TcShared) <= 2048, "operands start 2048 bytes into shared memory");

// 16 columns of this thread's lane from tensor memory, and 8 + 8 to it.
DLLM_DEV void tmem_ld16(uint32_t addr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(addr));
}
DLLM_DEV void tmem_st16(uint32_t addr, const uint32_t (&h)[8], const uint32_t (&l)[8]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::"r"(h[0]),
      "r"(h[1]), "r"(h[2]), "r"(h[3]), "r"(h[4]), "r"(h[5]), "r"(h[6]), "r"(h[7]), "r"(l[0]), "r"(l[1]), "r"(l[2]), "r"(l[3]),
      "r"(l[4]), "r"(l[5]), "r"(l[6]), "r"(l[7]), "r"(addr)
      : "memory");
}
DLLM_DEV float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// Two values of p, below 2^16, as two fp16 terms each: the high one cut to 11 bits (its cut is
// exact in fp16; below 2^-14 it rounds, by 2^-25 at most), the low one rounded.
DLLM_DEV void split_p(float x, float y, uint32_t& h, uint32_t& l) {
  const float a = __uint_as_float(__float_as_uint(x) & 0xffffe000u), b = __uint_as_float(__float_as_uint(y) & 0xffffe000u);
  h = pack_f16(a, b);
  l = pack_f16(x - a, y - b);
}
DLLM_DEV void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

// The MMA's shared-memory descriptors (tc.cuh) as two words: the upper one is the same for all
// operands here, and the lower one moves by constants (2% of a long chunk's time against 64-bit
// values built anew).
constexpr uint32_t kDescHigh = 64u | 1u << 14 | 2u << 29;
DLLM_DEV uint32_t desc_low(const void* tile, uint32_t leading) { return (smem_u32(tile) & 0x3FFFFu) >> 4 | leading << 16; }
DLLM_DEV void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 x, y;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "mov.b64 x, {%1, %5};\n\t"
      "mov.b64 y, {%2, %5};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"(accumulate), "n"(kDescHigh));
}
DLLM_DEV void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 y;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "mov.b64 y, {%2, %5};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %3, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"(accumulate), "n"(kDescHigh));
}

template <int KIND, int HD>
__global__ void __launch_bounds__(kTcThreads, 1) rows_tc_kernel(const __grid_constant__ RowsKernelArgs P) {
  using T = TcTile<KIND, HD>;
  constexpr int BN = T::BN, BOX = T::BOX;
  extern __shared__ __align__(1024) unsigned char base[];
  __shared__ __align__(8) TcShared sh;
  const RowsAttnArgs& a = P.a;
  asm volatile("griddepcontrol.launch_dependents;");  // the join may be scheduled; it waits for this grid's end

  // the warp's number as a value that is the same in all its lanes by construction
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  unsigned char* sQ = base;  // [tile][term][box][128 rows][128 bytes]
  unsigned char* ring = base + 4 * T::kTile;

  // number of the block that starts at slot s0 among all (KV head, block) pairs
  auto unit_of = [&](const RowsTile& k, int s0) {
    const RowsView all(k.t0, k.t0 + k.m - 1, a.window, a.sinks, BN);
    const int blk = s0 / BN;
    return P.unit0[k.i] + k.head * all.nb + (blk >= all.first ? blk - all.first + all.nsink : blk);
  };

  if (tid == 0) {
    for (int s = 0; s < T::kRing; ++s) mbar_init(&sh.empty[s], 1);
    for (int i = 0; i < T::kTurns; ++i) mbar_init(&sh.pv_ready[i], 128 + 1), mbar_init(&sh.ok_ready[i], 1 + 1);
    for (int w = 0; w < 2; ++w) mbar_init(&sh.s_full[w], 1), mbar_init(&sh.o_full[w], 1);
    mbar_init(&sh.p1_ready, 128), mbar_init(&sh.o1_done, 1);
    for (int w = 0; w < 2; ++w) mbar_init(&sh.q_ready[w], 128);
    mbar_init(&sh.idle, 1);
    mbar_arrive(&sh.ok_ready[0]);  // the first scores wait for no O
    sh.abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kTcSoftWarps) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem)), "r"(512u));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, sh.tmem, 0);

  if (warp >= kTcSoftWarps) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    if (warp == kTcSoftWarps && lane == 0) {
      asm volatile("griddepcontrol.wait;" ::: "memory");  // the blocks are there
      // ---- producer: tile t is K of block t / 2 (even) or V. It reports to the barriers that the
      // first tile's MMAs wait for: ok_ready of the block (K), pv_ready (V). A barrier's earlier turn, 2
      // kTurns >= kRing tiles before, has ended: the stage's earlier tile came later, and is used up.
      int sent = 0;
      const unsigned char* planes = static_cast<const unsigned char*>(a.planes);
      auto bar = [&](int t) { return t & 1 ? &sh.pv_ready[t / 2 % T::kTurns] : &sh.ok_ready[t / 2 % T::kTurns]; };
      rows_segments(P, kTcTileRows, BN, [&](const RowsTile& k, int b0, int b1, bool) {
        for (int b = 2 * b0; b < 2 * b1; ++b) {
          const int t = sent, s = t % T::kRing;
          // nothing is loaded over memory that may still be read
          if (!wait_phase(&sh.empty[s], ((uint32_t)(t / T::kRing) & 1u) ^ 1u, &sh.abort)) return;
          mbar_expect_tx(bar(t), T::kTile);
          bulk_load(ring + s * T::kTile, planes + ((size_t)unit_of(k, k.v.slot0(b / 2, BN)) * 2 + (b & 1)) * T::kTile, T::kTile, bar(t));
          sent = t + 1;
        }
      });
      // whatever happened to the others, the copies under way land before the CTA ends
      for (int t = max(0, sent - T::kRing); t < sent; ++t) mbar_wait(bar(t), (uint32_t)(t / 2 / T::kTurns) & 1u);
    } else if (warp == kTcSoftWarps + 1) {
      // ---- MMA issuer. The whole warp runs the loop and one elected lane issues, so that the operands
      // stay in uniform registers. Little more than one MMA queues up behind the running one, and a wait
      // costs 100 to 200 cycles while shared memory serves the operands, even where nothing is left to wait
      // for: so there is one for each of the four products of a block, and no more. (A warp per tile
      // was slower: both tiles' MMAs then ran, and both softmaxes waited, at the same time.)
      const uint32_t leader = elect_one();
      const uint32_t idesc = (1u << 4) | ((uint32_t)(128 >> 4) << 24);                // fp32 += fp16 x fp16, M = 128
      const uint32_t id_s = idesc | ((uint32_t)(128 >> 3) << 17);                     // N = 128 rows of K, K-major
      const uint32_t id_half = idesc | ((uint32_t)(64 >> 3) << 17);                   // the first 64 of them
      const uint32_t id_o = idesc | ((uint32_t)(HD >> 3) << 17) | (1u << 16);         // N = dims, B with N contiguous
      constexpr uint32_t kTile16 = T::kTile >> 4, kBox16 = T::kBox >> 4;
      const uint32_t q_low = desc_low(sQ, 1u), k_low = desc_low(ring, 1u), v_low = desc_low(ring, T::kBox >> 4);
      int tiles = 0;
      auto scores = [&](int w, int n) {
        tc_fence_after();
        if (leader) {
          const int s = 2 * n % T::kRing;
          const uint32_t d = tmem + (uint32_t)w * 128, q = q_low + (uint32_t)w * (2 * kTile16), kb = k_low + (uint32_t)s * kTile16;
          // the low term of q first; with two planes of K it comes second, into their half
#pragma unroll
          for (int term = 0; term < 2; ++term) {
            const uint32_t qt = q + (T::kPlanes == 1 ? 1 - term : term) * kTile16;
#pragma unroll
            for (int x = 0; x < BOX; ++x)
#pragma unroll
              for (int kk = 0; kk < 4; ++kk) {
                const uint32_t at = x * kBox16 + 2 * kk;
                if (T::kPlanes == 2 && term == 1) mma_ss(d + 64, qt + at, kb + at, id_half, 1u);
                else mma_ss(d, qt + at, kb + at, id_s, (uint32_t)(term || x || kk));
              }
          }
          umma_commit(&sh.s_full[w]);
          if (w == tiles - 1) umma_commit(&sh.empty[s]);
        }
        __syncwarp();
      };
      auto output = [&](int w, int n) {
        tc_fence_after();
        if (leader) {
          const int s = (2 * n + 1) % T::kRing;
          const uint32_t p = tmem + (uint32_t)w * 128, d = p + 256u, vb = v_low + (uint32_t)s * kTile16;
          // products (term of p, plane of V), the smallest first
#pragma unroll
          for (int i = 0; i < T::kPlanes + 1; ++i) {
            const int low = i == 0, plane = T::kPlanes == 2 && i == 1;
#pragma unroll
            for (int ks = 0; ks < BN / 16; ++ks)  // 16 slots: 2048 bytes on
              mma_ts(d, p + 16u * ks + 8u * low, vb + (plane * (BN * 128) + ks * 2048) / 16, id_o, (uint32_t)(i || ks));
          }
          umma_commit(w ? &sh.o1_done : &sh.ok_ready[(n + 1) % T::kTurns]);
          umma_commit(&sh.o_full[w]);
          if (w == tiles - 1) umma_commit(&sh.empty[s]);
        }
        __syncwarp();
      };
      auto turn = [&](int n) { return (uint32_t)(n / T::kTurns) & 1u; };
      // blocks of the CTA so far, those with a second tile, and segments of each tile
      int n = 0, n1 = 0;
      uint32_t segments[2] = {0u, 0u};
      rows_segments(P, kTcTileRows, BN, [&](const RowsTile& k, int b0, int b1, bool) {
        tiles = k.R - k.r0 > 128 ? 2 : 1;
        wait_phase(&sh.ok_ready[n % T::kTurns], turn(n), &sh.abort);
        for (int w = 0; w < tiles; ++w) {
          wait_phase(&sh.q_ready[w], segments[w]++ & 1u, &sh.abort);  // (and the output before has been read)
          scores(w, n);
        }
        for (int b = b0; b < b1; ++b, ++n) {
          const bool more = b + 1 < b1;
          // P is there (and so O of the block before has been read), and V; the next scores replace P
          wait_phase(&sh.pv_ready[n % T::kTurns], turn(n), &sh.abort);
          output(0, n);
          if (more) {
            wait_phase(&sh.ok_ready[(n + 1) % T::kTurns], turn(n + 1), &sh.abort);
            scores(0, n + 1);
          }
          if (tiles == 2) {
            wait_phase(&sh.p1_ready, (uint32_t)n1 & 1u, &sh.abort);
            output(1, n);
            if (more) {
              wait_phase(&sh.o1_done, (uint32_t)n1 & 1u, &sh.abort);
              scores(1, n + 1);
            }
            ++n1;
          }
        }
      });
      // nothing of this warp's is under way when the tensor memory is freed
      if (leader) umma_commit(&sh.idle);
      __syncwarp();
      mbar_wait(&sh.idle, 0u);
    }
    __syncwarp();
  } else {
    // ---- softmax: group w, one row of its tile per thread
    asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    const int w = warp >> 2, me = tid & 127;
    const uint32_t lanes = tmem + (uint32_t)w * 128 + ((uint32_t)((warp & 3) * 32) << 16);
    unsigned char* tile = sQ + w * 2 * T::kTile;
    int done = 0;  // blocks of this tile's (of the first tile's: of the CTA)
    rows_segments(P, kTcTileRows, BN, [&](const RowsTile& k, int b0, int b1, bool first_segment) {
      const int nb = b1 - b0, r0 = k.r0 + w * 128;
      if (r0 >= k.R) return;
      // ---- q: rows scaled so that the softmax is in powers of two, each divided by a power of two
      // next to its largest element, as two fp16 terms. Rows behind the last one are zero.
      {
        constexpr int C = HD / 8, kPass = 128 / C, kBatch = 8;  // C threads per row
        const int c = me % C;
#pragma unroll 1
        for (int r1 = me / C; r1 < 128; r1 += kPass * kBatch) {
          float x[kBatch][8];
#pragma unroll
          for (int u = 0; u < kBatch; ++u) {
            const int r = r0 + r1 + u * kPass;
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
            unsigned char* p = tile + (c / 8) * T::kBox + row * 128 + (((c & 7) ^ (row & 7)) << 4);
            *reinterpret_cast<uint4*>(p) = make_uint4(h[0], h[1], h[2], h[3]);
            *reinterpret_cast<uint4*>(p + T::kTile) = make_uint4(l[0], l[1], l[2], l[3]);
            if (c == 0) sh.back[w * 128 + row] = power_of_two(ex - 14);
          }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // q is read by the MMA
        mbar_arrive(&sh.q_ready[w]);
        asm volatile("bar.sync %0, 128;" ::"r"(1 + w) : "memory");  // `back` is there
      }
      asm volatile("griddepcontrol.wait;" ::: "memory");  // the blocks' factors are there
      const int slot = k.slot_of(r0 + me);
      float o[HD], m = -INFINITY, l = 0.f, unit = 0.f;
#pragma unroll
      for (int d = 0; d < HD; ++d) o[d] = 0.f;
      const float back = sh.back[w * 128 + me];
      // the rows of this tile see slots up to p0 at least, and from p1 - window on
      const int p0 = k.t0 + r0 / k.G, p1 = k.t0 + (min(r0 + 128, k.R) - 1) / k.G;
      const uint32_t* info = reinterpret_cast<const uint32_t*>(a.info);  // K's low, V's high
      int s0 = k.v.slot0(b0, BN);
      uint32_t next = info[unit_of(k, s0)];
      for (int n = 0; n < nb; ++n, ++done) {
        const uint32_t now = next;
        const int s_now = s0;
        if (n + 1 < nb) {
          s0 = k.v.slot0(b0 + n + 1, BN);
          next = info[unit_of(k, s0)];
        }
        float f = fmaxf(back * power_of_two((int)(now & 255u) - 14), 1.175494351e-38f);  // (-inf times 0 would be NaN)
        const bool edge = s_now + BN - 1 > p0 || (s_now <= p1 - a.window && s_now + BN > a.sinks);
        // column c of the block is visible where c <= last and (c >= first or c < sink)
        const int last = slot - s_now, first = last >= a.window ? last - a.window + 1 : 0, sink = a.sinks - s_now;
        wait_phase(&sh.s_full[w], (uint32_t)done & 1u, &sh.abort);
        tc_fence_after();
        // ---- wide blocks, 8 columns at a time: what the MMA left of them (two parts of it where K is two
        // planes), and the powers of their slots
        auto exps = [&](int v) {
          return reinterpret_cast<const uint2*>(a.exps + (2 * (size_t)unit_of(k, s_now) + v) * kTcExps);
        };
        auto exp_at = [](uint2 x, int e) { return (int)((e < 4 ? x.x : x.y) >> (e % 4 * 8) & 255u); };
        auto fetch8 = [&](int c, uint32_t(&u)[8], uint32_t(&z)[8]) {
          tmem_ld8(lanes + (uint32_t)c, u);
          if constexpr (T::kPlanes == 2) tmem_ld8(lanes + (uint32_t)(64 + c), z);
          tmem_ld_wait();
        };
        auto put8 = [&](int c, const uint32_t(&u)[8]) {
          tmem_st8(lanes + (uint32_t)c, u);
          if constexpr (T::kPlanes == 2) {
            const uint32_t zero[8] = {0u, 0u, 0u, 0u, 0u, 0u, 0u, 0u};
            tmem_st8(lanes + (uint32_t)(64 + c), zero);
          }
        };
        if (__builtin_expect((now & kTcWide) != 0u, 0)) {  // the scores themselves over it
          const uint2* own = exps(0);
#pragma unroll 1
          for (int c = 0; c < BN; c += 8) {
            uint32_t u[8], z[8];
            const uint2 ex = own[c / 8];
            fetch8(c, u, z);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              float y = __uint_as_float(u[e]);
              if constexpr (T::kPlanes == 2) y += __uint_as_float(z[e]);
              u[e] = __float_as_uint(y * fmaxf(back * power_of_two(exp_at(ex, e) - 14), 1.175494351e-38f));
            }
            put8(c, u);
          }
          tmem_st_wait();
          f = 1.f;
        }
        // ---- the largest score; hidden ones are at -inf here and below
        uint32_t ua[32], ub[32];
        float x = -INFINITY, x1 = x, x2 = x, x3 = x;
        auto most = [&](const uint32_t(&u)[32]) {
#pragma unroll
          for (int e = 0; e < 32; e += 8) {
            x = max3(x, __uint_as_float(u[e]), __uint_as_float(u[e + 1]));
            x1 = max3(x1, __uint_as_float(u[e + 2]), __uint_as_float(u[e + 3]));
            x2 = max3(x2, __uint_as_float(u[e + 4]), __uint_as_float(u[e + 5]));
            x3 = max3(x3, __uint_as_float(u[e + 6]), __uint_as_float(u[e + 7]));
          }
        };
        // bit e: column c + e is visible (no branches: they would part the rows of a warp)
        auto below = [](int n) { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1; };
        auto visible = [&](int c) { return below(last - c + 1) & (~below(first - c) | below(sink - c)); };
        if (__builtin_expect(edge, 0)) {
#pragma unroll 1
          for (int c = 0; c < BN; c += 16) {
            uint32_t u[16], z[16];
            tmem_ld16(lanes + (uint32_t)c, u);
            if constexpr (T::kPlanes == 2) tmem_ld16(lanes + (uint32_t)(64 + c), z);
            const uint32_t see = visible(c);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              float y = __uint_as_float(u[e]);
              if constexpr (T::kPlanes == 2) y += __uint_as_float(z[e]);
              x = fmaxf(x, see >> e & 1 ? y : -INFINITY);
            }
          }
        } else if constexpr (T::kPlanes == 2) {
#pragma unroll
          for (int c = 0; c < BN; c += 32) {
            tmem_ld32(lanes + (uint32_t)c, ua);
            tmem_ld32(lanes + (uint32_t)(64 + c), ub);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 32; ++e) ua[e] = __float_as_uint(__uint_as_float(ua[e]) + __uint_as_float(ub[e]));
            most(ua);
          }
        } else {
          tmem_ld32(lanes, ua);
#pragma unroll
          for (int c = 0; c < BN; c += 64) {
            tmem_ld_wait();
            tmem_ld32(lanes + (uint32_t)(c + 32), ub);
            most(ua);
            tmem_ld_wait();
            if (c + 64 < BN) tmem_ld32(lanes + (uint32_t)(c + 64), ua);
            most(ub);
          }
        }
        x = fmaxf(max3(x, x1, x2), x3) * f;
        // p is 2^(x - m + 8) with scores x up to m + 7: m is the row's maximum at a time, and moves late (with
        // l and o) only when a score exceeds that. (m + 7 could round up, and p then leave fp16's range.)
        if (__any_sync(0xffffffffu, x - m > 7.f)) {
          const float to = fmaxf(m, x), g = to == -INFINITY ? 1.f : ex2(m - to);
          m = to, l *= g;
#pragma unroll
          for (int d = 0; d < HD; ++d) o[d] *= g;
        }
        const float base = m == -INFINITY ? 0.f : m;
        const float shift = 8.f - base + base > 15.f ? -base : 8.f - base;  // (8 - m may round to 16 - m)
        // V's factor; a row that sees nothing of the block keeps the unit of its o.
        float fv = x == -INFINITY ? unit : power_of_two((int)(now >> 16 & 255u) - 14);
        // In a wide block it is the largest of the slots that the row sees: p takes the others' powers
        // relative to it, in its exponent, after its sum.
        if (__builtin_expect((now >> 16 & kTcWide) != 0u, 0)) {
          const uint2* own = exps(1);
          int top = 15;
#pragma unroll 1
          for (int c = 0; c < BN; c += 8) {
            uint32_t u[8], z[8];
            const uint2 ex = own[c / 8];
            const uint32_t see = visible(c);
            fetch8(c, u, z);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              float y = __uint_as_float(u[e]);
              if constexpr (T::kPlanes == 2) y += __uint_as_float(z[e]);
              y = fmaf(y, f, shift);
              if (see >> e & 1) top = max(top, exp_at(ex, e));
              l += see >> e & 1 ? ex2(y) : 0.f;
            }
          }
#pragma unroll 1
          for (int c = 0; c < BN; c += 8) {
            uint32_t u[8], z[8];
            const uint2 ex = own[c / 8];
            fetch8(c, u, z);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              float y = __uint_as_float(u[e]);
              if constexpr (T::kPlanes == 2) y += __uint_as_float(z[e]);
              u[e] = __float_as_uint(fmaf(y, f, (float)(exp_at(ex, e) - top)));
            }
            put8(c, u);
          }
          tmem_st_wait();
          f = 1.f;
          if (x != -INFINITY) fv = power_of_two(top - 14);
        }
        // ---- p over the scores, 32 columns of tensor memory at a time (32 scores, or 16 and their
        // second parts): while the exponentials of some are under way, the next ones land. A loop, not
        // unrolled: the code of both groups has to stay in the instruction cache. (And no decision inside:
        // with a vote per 16 columns they took 3700 cycles per 128 columns, two warps on a scheduler, and
        // take 2800, 2050 of which are the exponentials.)
        float sum = 0.f;
        auto fetch = [&](int i) {
          uint32_t(&u0)[16] = reinterpret_cast<uint32_t(&)[16]>(ua[0]);
          uint32_t(&u1)[16] = reinterpret_cast<uint32_t(&)[16]>(ua[16]);
          if constexpr (T::kPlanes == 1) tmem_ld16(lanes + (uint32_t)(32 * i), u0), tmem_ld16(lanes + (uint32_t)(32 * i + 16), u1);
          else tmem_ld16(lanes + (uint32_t)(16 * i), u0), tmem_ld16(lanes + (uint32_t)(64 + 16 * i), u1);
        };
        constexpr int kStep = 32 / T::kPlanes;
        fetch(0);
#pragma unroll 1
        for (int i = 0; i < 4; ++i) {
          float y[kStep];
          tmem_ld_wait();
#pragma unroll
          for (int e = 0; e < kStep; ++e) {
            // the same sum as above: f is a power of two, so the largest score's p is 2^8 at any size of it
            float u = __uint_as_float(ua[e]);
            if constexpr (T::kPlanes == 2) u += __uint_as_float(ua[16 + e]);
            y[e] = fmaf(u, f, shift);
          }
          if (i < 3) fetch(i + 1);
          if (__builtin_expect(edge, 0)) {
            const uint32_t see = visible(i * kStep);
#pragma unroll
            for (int e = 0; e < kStep; ++e) y[e] = see >> e & 1 ? y[e] : -INFINITY;
          }
#pragma unroll
          for (int c = 0; c < kStep; c += 16) {
            uint32_t ph[8], pl[8];
            float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const float q0 = ex2(y[c + 2 * e]), q1 = ex2(y[c + 2 * e + 1]);
              s[e % 2 * 2] += q0, s[e % 2 * 2 + 1] += q1;
              split_p(q0, q1, ph[e], pl[e]);
            }
            tmem_st16(lanes + (uint32_t)(i * kStep + c), ph, pl);
            sum += (s[0] + s[1]) + (s[2] + s[3]);
          }
        }
        l += now >> 16 & kTcWide ? 0.f : sum;
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(w ? &sh.p1_ready : &sh.pv_ready[done % T::kTurns]);
        // o is in units of `unit`, a power of two that only grows
        float lift = 1.f, drop = 1.f;
        if (fv != unit) {
          const float to = fmaxf(fv, unit);
          lift = unit / to, drop = fv / to, unit = to;
        }
        const bool drops = __any_sync(0xffffffffu, drop != 1.f);
        wait_phase(&sh.o_full[w], (uint32_t)done & 1u, &sh.abort);
        tc_fence_after();
        const uint32_t from = lanes + 256u;
        auto take = [&](int d, uint32_t(&v)[32]) {
          if (__builtin_expect(drops, 0)) {
#pragma unroll
            for (int e = 0; e < 32; ++e) v[e] = __float_as_uint(__uint_as_float(v[e]) * drop);
          }
#pragma unroll
          for (int e = 0; e < 32; ++e) o[d + e] = fmaf(o[d + e], lift, __uint_as_float(v[e]));
        };
        tmem_ld32(from, ua);
#pragma unroll
        for (int d = 0; d < HD; d += 64) {
          tmem_ld_wait();
          tmem_ld32(from + (uint32_t)(d + 32), ub);
          take(d, ua);
          tmem_ld_wait();
          if (d + 64 < HD) tmem_ld32(from + (uint32_t)(d + 64), ua);
          take(d + 32, ub);
        }
        tc_fence_before();
        if (now >> 16 & kTcBad) {
#pragma unroll 1
          for (int c = 0; c < BN; ++c) {
            if (!(c <= last && (c >= first || c < sink))) continue;
            const size_t at = a.pages.row(k.seq, s_now + c, k.head);
#pragma unroll
            for (int d = 0; d < HD; d += 8) {
              float v[8];
              load8<KIND, HD>(a.vc, a.vs, at, d / 8, v);
#pragma unroll
              for (int e = 0; e < 8; ++e)
                if (!is_finite(v[e])) o[d + e] += v[e];
            }
          }
        }
      }
      // ---- results. Every MMA of this tile has completed (the group waited for its last O), so they pass
      // through q's memory, and rows leave whole.
      const bool whole = b0 == 0 && b1 == k.v.nb;
      const size_t part = ((size_t)blockIdx.x * 2 + !first_segment) * kTcTileRows + w * 128;
      const float scale = whole ? unit / l : unit;
      if (!whole && r0 + me < k.R) *reinterpret_cast<float2*>(a.part_ml + (part + me) * 2) = make_float2(m, l);
      constexpr int C4 = HD / 4;
      float4* stage = reinterpret_cast<float4*>(tile);
#pragma unroll
      for (int c = 0; c < C4; ++c)
        stage[me * C4 + (c ^ (me & (C4 - 1)))] =
            make_float4(o[4 * c] * scale, o[4 * c + 1] * scale, o[4 * c + 2] * scale, o[4 * c + 3] * scale);
      asm volatile("bar.sync %0, 128;" ::"r"(1 + w) : "memory");
      if (!sh.abort) {
        const int c = me % C4, rows = min(128, k.R - r0);
#pragma unroll 4
        for (int row = me / C4; row < rows; row += 128 / C4) {
          const float4 v = stage[row * C4 + (c ^ (row & (C4 - 1)))];
          float* to = whole ? a.out + ((size_t)k.row0 * a.nq + k.place(r0 + row, a.nq)) * HD : a.part_o + (part + row) * HD;
          reinterpret_cast<float4*>(to)[c] = v;
        }
      }
      asm volatile("bar.sync %0, 128;" ::"r"(1 + w) : "memory");  // the next q may come
    });
  }
  tc_fence_before();
  __syncthreads();
  if (tid == 0 && sh.abort) atomicExch(a.err, kErrRowsWait);
  if (warp == kTcSoftWarps) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u));
  }
}

// Shares below this many blocks are not worth a CTA of their own (its start, a partial result and
// the join take about as long as two blocks).
constexpr int kTcLeastShare = 2;

template <int KIND, int HD>
cudaError_t launch(const RowsAttnArgs& a, const RowsBatch& b, int sms, int* launches, cudaStream_t st) {
  using T = TcTile<KIND, HD>;
  RowsKernelArgs P;
  const RowsPlan plan = rows_plan(a, b, kTcTileRows, T::BN, sms, kTcLeastShare, 2, &P);
  P.a.exps = static_cast<unsigned char*>(a.planes) + (size_t)plan.units * 2 * T::kTile;
  P.a.info = reinterpret_cast<uint16_t*>(P.a.exps + (size_t)plan.units * 2 * kTcExps);
  rows_planes_kernel<KIND, HD><<<2 * plan.units, kPlaneThreads<KIND, HD>, 0, st>>>(P);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  e = launch_early(rows_tc_kernel<KIND, HD>, plan.ctas, kTcThreads, T::kSmem, st, P);
  *launches += 2;
  return e != cudaSuccess ? e : rows_join(P, plan, kTcTileRows, T::BN, HD, launches, st);
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

cudaError_t launch_rows_tc(const RowsAttnArgs& a, const RowsBatch& b, int kind, int hd, int sms, int* launches,
                           cudaStream_t st) {
  switch (kind) {
    case kKvF32: return hd == 64 ? launch<kKvF32, 64>(a, b, sms, launches, st) : launch<kKvF32, 128>(a, b, sms, launches, st);
    case kKvBf16: return hd == 64 ? launch<kKvBf16, 64>(a, b, sms, launches, st) : launch<kKvBf16, 128>(a, b, sms, launches, st);
    default: return hd == 64 ? launch<kKv4, 64>(a, b, sms, launches, st) : launch<kKv4, 128>(a, b, sms, launches, st);
  }
}

}  // namespace dllm
