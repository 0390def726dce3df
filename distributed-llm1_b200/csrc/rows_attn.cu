// rows_attn.cu — attention of a batch of rows over a paged cache, few rows per sequence.
//
// A row at cache slot p sees the slots s <= p with s > p - window or s < sinks:
//   out = sum_s p_s v_s,  p_s = exp(q . k_s / sqrt(hd) - max) / sum
// The m rows of a sequence and the G query heads of a KV head make m G rows that share one
// pass over that head's K and V; the softmax runs online over blocks of slots, blocks that
// no row of the tile sees are not read, and the blocks of a tile are split over CTAs whose
// partial results a second kernel joins.
//
// Precision. q, p and the outputs are fp32. bf16 and fp32 caches: q and p are cut into three
// bf16 or two tf32 terms (tree_attn.cu has the reasons). 4-bit rows, value = middle + scale *
// (code - 8) with middle = minimum + 8 scale:
//   q . k = sum over groups of 32 dims of scale * (q . (code - 8)) + middle * (sum of q)
//   o     = sum over slots of (p scale) (code - 8), + sum over slots of p middle
// (With the minima and the codes themselves both sums are far larger than what they add up to:
// over 8000 slots the outputs were off by 8e-6, and are by 7e-7.) Codes are exact in any 16-bit
// type, and the other operand runs as two fp16 terms (22 bits) of fp32 values brought into fp16's
// range by a power of two: a row of q by one next to its largest element, p scale by one next to
// the block's largest scale. A pair of codes becomes fp16 as (nibbles | bits of 1024) - 1032; the
// odd nibbles of a byte stay where they are, as 16 times their codes, and what they meet is a
// sixteenth. (The nibbles alone, read as fp16, are code * 2^-24, but the tensor core aligns such
// subnormal products by their exponents, 10 bits above their leading ones, and the sums lose as
// many: 4e-6 over 9 slots.) p meets the middles in bf16 terms, three of p and two of them.
//
// Work split. A CTA has 8 warps and takes 16 WR rows of one (sequence, KV head): WR warps
// side by side in rows, 8 / WR of them in slots, each with a maximum, sum and output of its
// own, joined at the end. K and V blocks come through a cp.async ring; slots behind the
// tile's last row are zero-filled, never read. Sequences and heads of any lengths are cut into
// equal shares for one wave of CTAs (rows_plan).
//
// Up to 8 rows (WR = 0: decode steps) the products' 16 rows would be half empty. There o is
// computed transposed, V^T (p^T): the 8 rows are the products' narrow side, what a thread holds of
// row g of the scores is what the second operand wants, and scaling, cutting and accumulating p
// and o take half the instructions and registers, so that two CTAs share an SM. In the scores
// the second terms of q take rows 8 to 15: one product instead of two. A warp copies the slots that it
// works on itself, without barriers in the loop.
//
// What bounds it. 24 sequences of 2000 to 4000 slots (3043 on average), 2 KV heads of 128, fp32: 41 us, 3.7
// TB/s; 64 of 4000 to 8000 (6032 on average) in 4 bits: 63 us, 2 TB/s, where a warp spends 1200 instructions
// per 32 slots, about as many each on the integer and the floating-point pipe (unpacking codes, cutting
// p, scales), and 70 MMAs.
#include "rows_attn.cuh"

#include <algorithm>
#include <type_traits>
#include <vector>

#include "mma_sync.cuh"
#include "rows_attn_tc.cuh"

namespace dllm {
namespace {

constexpr int kThreads = 256;
constexpr float kNegInf = -INFINITY;

DLLM_DEV void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Nibbles 0 and 4 of u, less 8, as packed fp16, and 16 times nibbles 1 and 5, less 8. (Small whole numbers
// as the low bits of a float whose unit they are, a well-known conversion.)
DLLM_DEV uint32_t codes_f16(uint32_t u) {
  uint32_t r;
  asm("{\n\t.reg .b32 t;\n\tlop3.b32 t, %1, 0x000f000f, 0x64006400, 0xea;\n\tsub.rn.f16x2 %0, t, %2;\n\t}"
      : "=r"(r)
      : "r"(u), "r"(0x64086408u));
  return r;
}
DLLM_DEV uint32_t codes16_f16(uint32_t u) {
  uint32_t r;
  asm("{\n\t.reg .b32 t;\n\tlop3.b32 t, %1, 0x00f000f0, 0x64006400, 0xea;\n\tsub.rn.f16x2 %0, t, %2;\n\t}"
      : "=r"(r)
      : "r"(u), "r"(0x64806480u));
  return r;
}
DLLM_DEV void cp8_zfill(uint32_t dst, const void* src, bool real) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst), "l"(src), "r"(real ? 8 : 0) : "memory");
}

// Tile shapes. SN: slots of a block that one warp takes; BN: slots of a block. The ring
// depth is what fits beside the q tile in 227 KB, four at most.
template <int KIND, int HD, int WR>
struct Tile {
  static constexpr bool kF32 = KIND == kKvF32, kQ4 = KIND == kKv4, kNarrow = WR == 0;
  static constexpr int WS = kNarrow ? 8 : 8 / WR;
  static constexpr int SN = kF32 ? (kNarrow ? 8 : 8 * WR) : WR == 1 || (kNarrow && !kQ4) ? 16 : 32;
  static constexpr int BN = SN * WS;
  static constexpr int RT = kNarrow ? 8 : 16 * WR;
  static constexpr int kRowBytes = KvRow<KIND, HD>::kBytes;
  static constexpr int kPairBytes = KvRow<KIND, HD>::kPairs * 4;
  static constexpr int kChunks = kRowBytes / 16;
  static constexpr int kRows = BN * kRowBytes, kTileBytes = kRows + BN * kPairBytes;  // one of K, V
  static constexpr int kCtas = kNarrow && kQ4 ? 2 : 1;  // per SM
  static constexpr int kQRows = kNarrow && !kF32 ? 16 : RT;
  // (wide 4-bit tiles keep q in registers)
  static constexpr int kQBytes = kQ4 ? (kNarrow ? HD * 32 : 0) : kQRows * HD * (kF32 ? 4 : kNarrow ? 4 : 6);
  static constexpr int kPad = HD + 4;
  static constexpr int kMergeBytes = WS * RT * (kPad + 2) * 4;
  static constexpr int kFit = ((kCtas == 2 ? 112 : 225) * 1024 - kQBytes) / (2 * kTileBytes);
  static constexpr int kStages = kFit > 4 ? 4 : kFit;
  static constexpr int kRing = kStages * 2 * kTileBytes;
  static constexpr int kSmem = kQBytes + (kRing > kMergeBytes ? kRing : kMergeBytes);
  static_assert(kStages >= 2 && kCtas * (kSmem + 1024) <= 228 * 1024, "shared memory");
  static_assert(BN % 32 == 0, "a page lookup serves 32 slots");
};

// Where 16-byte chunk c of a 4-bit K or V row lies: K is read by 8 slots at once (a word of one
// chunk each), V by 4, both without bank conflicts.
template <int HD, bool V>
DLLM_DEV uint32_t at4(int row, int c) {
  if constexpr (HD == 128)
    return row * 64 + ((V ? c ^ (row >> 1 & 1) : c ^ (row >> 1 & 3)) << 4);
  else
    return row * 32 + ((V ? c : c ^ (row >> 2 & 1)) << 4);
}

template <int KIND, int HD, int WR>
__global__ void __launch_bounds__(kThreads, Tile<KIND, HD, WR>::kCtas) rows_attn_kernel(const __grid_constant__ RowsKernelArgs P) {
  using T = Tile<KIND, HD, WR>;
  constexpr int SN = T::SN, BN = T::BN, WS = T::WS, RT = T::RT, NT = SN / 8, CH = T::kChunks, S = T::kStages;
  constexpr bool F32 = T::kF32, Q4 = T::kQ4, N8 = T::kNarrow;
  constexpr int NG = HD / kGroup4;  // 4-bit rows: groups
  extern __shared__ __align__(1024) unsigned char smem[];
  const RowsAttnArgs& a = P.a;
  launch_next_and_wait();
  const int window = a.window, sinks = a.sinks;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int wr = N8 ? 0 : warp % (N8 ? 1 : WR), ws = N8 ? warp : warp / (N8 ? 1 : WR);
  const int g = lane >> 2, t = lane & 3;
  unsigned char* sQ = smem;
  unsigned char* ring = smem + T::kQBytes;
  rows_segments(P, RT, BN, [&](const RowsTile& k, int b0, int b1, bool first_segment) {
    const int end = k.v.p1 + 1;

    // ---- K/V blocks through the ring. Pages hold at least 32 slots, so a block has BN / 32
    // page lookups at most, made one block ahead of the copies that need them. A narrow tile's
    // warps copy the slots that they work on themselves: one page each, and no barriers.
    const int* table = a.pages.table + (size_t)k.seq * a.pages.max_pages;
    const int log2_page = a.pages.log2_page, in_page = (1 << log2_page) - 1;
    const int wslot = ws * SN;  // first slot of this warp within a block
    const unsigned char *kc = static_cast<const unsigned char*>(a.kc), *vc = static_cast<const unsigned char*>(a.vc);
    constexpr int kPages = N8 ? 1 : BN / 32;
    int page[kPages];
    auto lookup = [&](int b) {
      const int s0 = k.v.slot0(b, BN);
#pragma unroll
      for (int i = 0; i < kPages; ++i) page[i] = __ldg(table + (min(s0 + (N8 ? wslot : 32 * i), end - 1) >> log2_page));
    };
    auto row_of = [&](int s0, int row) {
      int pg = page[0];
#pragma unroll
      for (int u = 1; u < kPages; ++u) pg = row >= 32 * u ? page[u] : pg;
      return (((size_t)pg * a.pages.kvh + k.head) << log2_page) + ((s0 + row) & in_page);
    };
    auto at_k = [](int row, int c) -> uint32_t {
      if constexpr (Q4) return at4<HD, false>(row, c);
      else return row * T::kRowBytes + ((c ^ (row & 7)) << 4);
    };
    auto at_v = [](int row, int c) -> uint32_t {
      if constexpr (Q4) return at4<HD, true>(row, c);
      else return row * T::kRowBytes + ((c ^ (row & 7)) << 4);
    };
    auto copy = [&](int b, int stage) {
      const int s0 = k.v.slot0(b, BN);
      const uint32_t dk = smem_addr(ring + stage * 2 * T::kTileBytes), dv = dk + T::kTileBytes;
      if constexpr (N8) {
        constexpr int kPass = 32 / CH > 0 ? 32 / CH : 1;  // slots per pass
        const size_t row0 = row_of(s0, wslot);
        const int c = lane % CH, left = end - (s0 + wslot);
#pragma unroll
        for (int i = 0; i < SN / kPass; ++i) {
          const int row = lane / CH + i * kPass;
          const size_t off = (row0 + row) * T::kRowBytes + c * 16;
          const bool real = row < left;
          cp16_zfill(dk + at_k(wslot + row, c), real ? kc + off : kc, real);
          cp16_zfill(dv + at_v(wslot + row, c), real ? vc + off : vc, real);
        }
        if constexpr (Q4) {
          static_assert(SN == 32, "a lane copies the pairs of one slot");
          const size_t off = (row0 + lane) * NG;
          const bool real = lane < left;
          const uint32_t at = T::kRows + (wslot + lane) * T::kPairBytes;
          if constexpr (HD == 128)
            cp16_zfill(dk + at, real ? a.ks + off : a.ks, real), cp16_zfill(dv + at, real ? a.vs + off : a.vs, real);
          else
            cp8_zfill(dk + at, real ? a.ks + off : a.ks, real), cp8_zfill(dv + at, real ? a.vs + off : a.vs, real);
        }
      } else {
        constexpr int kPass = kThreads / CH;  // slots per pass
        const int c = tid % CH;
#pragma unroll
        for (int i = 0; i < (BN + kPass - 1) / kPass; ++i) {
          const int row = tid / CH + i * kPass;
          if (BN % kPass && row >= BN) break;
          const size_t off = row_of(s0, row) * T::kRowBytes + c * 16;
          const bool real = s0 + row < end;
          cp16_zfill(dk + at_k(row, c), real ? kc + off : kc, real);
          cp16_zfill(dv + at_v(row, c), real ? vc + off : vc, real);
        }
        if constexpr (Q4) {
#pragma unroll
          for (int i = 0; i < (2 * BN + kThreads - 1) / kThreads; ++i) {
            const int at = tid + i * kThreads, row = at % BN;
            if (2 * BN % kThreads && at >= 2 * BN) break;
            const bool real = s0 + row < end;
            const uint32_t* src = at < BN ? a.ks : a.vs;
            const uint32_t dst = (at < BN ? dk : dv) + T::kRows + row * T::kPairBytes;
            if (real) src += row_of(s0, row) * NG;
            if constexpr (HD == 128) cp16_zfill(dst, src, real);
            else cp8_zfill(dst, src, real);
          }
        }
      }
    };
    lookup(b0);
#pragma unroll
    for (int s = 0; s < S - 1; ++s) {
      if (b0 + s < b1) {
        copy(b0 + s, s);
        lookup(min(b0 + s + 1, b1 - 1));
      }
      cp_commit();
    }

    // this thread's two rows of the tile
    const int ra = wr * 16 + g, rb = ra + 8;
    const int pa = k.slot_of(k.r0 + ra), pb = N8 ? -1 : k.slot_of(k.r0 + rb);

    // ---- the q tile, scaled by log2(e) / sqrt(hd) so that the softmax is in powers of two
    uint32_t qf[Q4 && !N8 ? HD / 16 : 1][2][4];  // 4-bit rows: A fragments of two fp16 terms
    uint4* qs = reinterpret_cast<uint4*>(sQ) + lane;  // of a narrow tile: [k step][lane]
    float qsum_a[Q4 ? NG : 1], qsum_b[Q4 ? NG : 1], back_a = 1.f, back_b = 1.f;
    if constexpr (Q4) {
      // lane t of a row holds dims 8t .. 8t + 7 of every group: a u32 of codes
      float xa[NG][8], xb[NG][8], ma = 0.f, mb = 0.f;
      const float* qa = a.q + ((size_t)k.row0 * a.nq + (pa < 0 ? 0 : k.place(k.r0 + ra, a.nq))) * HD + t * 8;
      const float* qb = a.q + ((size_t)k.row0 * a.nq + (pb < 0 ? 0 : k.place(k.r0 + rb, a.nq))) * HD + t * 8;
#pragma unroll
      for (int i = 0; i < NG; ++i)
#pragma unroll
        for (int e = 0; e < 8; e += 4) {
          const float4 z = make_float4(0.f, 0.f, 0.f, 0.f);
          const float4 fa = pa < 0 ? z : *reinterpret_cast<const float4*>(qa + i * kGroup4 + e);
          const float4 fb = pb < 0 ? z : *reinterpret_cast<const float4*>(qb + i * kGroup4 + e);
          xa[i][e] = fa.x, xa[i][e + 1] = fa.y, xa[i][e + 2] = fa.z, xa[i][e + 3] = fa.w;
          xb[i][e] = fb.x, xb[i][e + 1] = fb.y, xb[i][e + 2] = fb.z, xb[i][e + 3] = fb.w;
        }
#pragma unroll
      for (int i = 0; i < NG; ++i) {
        qsum_a[i] = qsum_b[i] = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          xa[i][e] *= a.scale_log2, xb[i][e] *= a.scale_log2;
          ma = fmaxf(ma, fabsf(xa[i][e])), mb = fmaxf(mb, fabsf(xb[i][e]));
          qsum_a[i] += xa[i][e], qsum_b[i] += xb[i][e];
        }
      }
#pragma unroll
      for (int w = 1; w < 4; w <<= 1) {
        ma = fmaxf(ma, __shfl_xor_sync(0xffffffffu, ma, w));
        mb = fmaxf(mb, __shfl_xor_sync(0xffffffffu, mb, w));
#pragma unroll
        for (int i = 0; i < NG; ++i) {
          qsum_a[i] += __shfl_xor_sync(0xffffffffu, qsum_a[i], w);
          qsum_b[i] += __shfl_xor_sync(0xffffffffu, qsum_b[i], w);
        }
      }
      // 2^e next to the largest element: the row divided by it, times 16, lies in [-32, 32] (dims that meet
      // 16 times their codes lack the 16). The exponent is kept where the factors are normal numbers.
      auto power = [](float m) { return min(max((int)(__float_as_uint(m) >> 23) & 0xff, 5), 253); };
      const int ea = power(ma), eb = power(mb);
      const float ia = power_of_two(258 - ea), ib = power_of_two(258 - eb);
      back_a = power_of_two(ea - 4), back_b = power_of_two(eb - 4);
#pragma unroll
      for (int i = 0; i < NG; ++i) qsum_a[i] *= ia, qsum_b[i] *= ib;
#pragma unroll
      for (int ks = 0; ks < HD / 16; ++ks) {
        const int i = ks / 2, d = (ks & 1) * 2;
        uint32_t f[2][4];
#pragma unroll
        for (int u = 0; u < 2; ++u) {  // dims d + u and d + u + 4: the two halves of a nibble pair
          const float ja = u ? ia * 0.0625f : ia, jb = u ? ib * 0.0625f : ib;
          split2_f16(xa[i][d + u] * ja, xa[i][d + u + 4] * ja, f[0][2 * u], f[1][2 * u]);
          split2_f16(xb[i][d + u] * jb, xb[i][d + u + 4] * jb, f[0][2 * u + 1], f[1][2 * u + 1]);
        }
        if constexpr (N8) {
          if (warp == ks % 8) qs[ks * 32] = make_uint4(f[0][0], f[1][0], f[0][2], f[1][2]);  // (all warps have it)
        } else {
#pragma unroll
          for (int term = 0; term < 2; ++term)
#pragma unroll
            for (int e = 0; e < 4; ++e) qf[ks][term][e] = f[term][e];
        }
      }
    } else {
      for (int i = tid; i < T::kQRows * HD / 4; i += kThreads) {
        const int row = i / (HD / 4), d = (i % (HD / 4)) * 4;
        const int r = k.r0 + row;
        float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
        if (row < RT && r < k.R) {
          f = *reinterpret_cast<const float4*>(a.q + ((size_t)k.row0 * a.nq + k.place(r, a.nq)) * HD + d);
          f.x *= a.scale_log2, f.y *= a.scale_log2, f.z *= a.scale_log2, f.w *= a.scale_log2;
        }
        if constexpr (F32) {
          *reinterpret_cast<float4*>(sQ + row * HD * 4 + (((d >> 2) ^ (row & 7)) << 4)) = f;
        } else {
          uint32_t h[2], m[2], l[2];
          split3(f.x, f.y, h[0], m[0], l[0]);
          split3(f.z, f.w, h[1], m[1], l[1]);
          unsigned char* p = sQ + row * HD * 2 + (((d >> 3) ^ (row & 7)) << 4) + (d & 4) * 2;
          if constexpr (N8) {  // rows 8 to 15: the second terms, and nothing beside the third ones
            if (row < RT) {
              *reinterpret_cast<uint2*>(p) = make_uint2(h[0], h[1]);
              *reinterpret_cast<uint2*>(p + RT * HD * 2) = make_uint2(m[0], m[1]);
            }
            *reinterpret_cast<uint2*>(p + T::kQRows * HD * 2) = make_uint2(l[0], l[1]);
            continue;
          }
          *reinterpret_cast<uint2*>(p) = make_uint2(h[0], h[1]);
          *reinterpret_cast<uint2*>(p + T::kQRows * HD * 2) = make_uint2(m[0], m[1]);
          *reinterpret_cast<uint2*>(p + 2 * T::kQRows * HD * 2) = make_uint2(l[0], l[1]);
        }
      }
    }

    // 4-bit rows: o of a group is in units of `unit` (a power of two, the same in the whole warp; dims of
    // odd nibbles of a byte: a sixteenth of it), and om is the middles' share, by group
    constexpr int NO = N8 ? HD / 16 : HD / 8;
    float o[NO][4], om[4] = {0.f, 0.f, 0.f, 0.f}, unit[Q4 ? NG : 1];
#pragma unroll
    for (int i = 0; i < (Q4 ? NG : 1); ++i) unit[i] = 0.f;
#pragma unroll
    for (int i = 0; i < NO; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[i][e] = 0.f;
    float ma = kNegInf, mb = kNegInf, la = 0.f, lb = 0.f;

    // the dim and the row of o[i][e] (4-bit rows have an order of their own)
    const int pc = N8 ? k.slot_of(k.r0 + 2 * t) : pa, pd = N8 ? k.slot_of(k.r0 + 2 * t + 1) : pb;
    auto dim_at = [&](int i, int e) { return N8 ? i * 16 + g + (e >> 1) * 8 : i * 8 + 2 * t + (e & 1); };
    auto second = [&](int e) { return N8 ? e & 1 : e >> 1; };  // of the thread's two rows

    // slot (within the block) of column c of this warp's score tile i. 4-bit rows: columns 2t and
    // 2t + 1 are slots t and t + 4, so that a lane's four slots of 16 are the ones whose V rows
    // it unpacks.
    auto slot_at = [&](int i, int e) {
      return Q4 ? wslot + i * 8 + t + (e & 1) * 4 : wslot + i * 8 + 2 * t + (e & 1);
    };

    if (N8) __syncthreads();  // q is there
    for (int b = b0; b < b1; ++b) {
      cp_wait<S - 2>();
      if (N8) __syncwarp();
      else __syncthreads();
      {
        const int next = b + S - 1;
        if (next < b1) {
          copy(next, (next - b0) % S);
          lookup(min(next + 1, b1 - 1));
        }
        cp_commit();
      }
      unsigned char* sK = ring + ((b - b0) % S) * 2 * T::kTileBytes;
      unsigned char* sV = sK + T::kTileBytes;
      const int s0 = k.v.slot0(b, BN);

      // ---- scores
      float sh[NT][4];
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) sh[i][e] = 0.f;
      if constexpr (Q4) {
#pragma unroll
        for (int gr = 0; gr < NG; ++gr) {
          uint32_t q[2][2][4];  // [k step][term]; a narrow tile has the second term in rows 8 to 15 of the first
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            if constexpr (N8) {
              const uint4 f = qs[(gr * 2 + u) * 32];
              q[u][0][0] = f.x, q[u][0][1] = f.y, q[u][0][2] = f.z, q[u][0][3] = f.w;
            } else {
#pragma unroll
              for (int e = 0; e < 8; ++e) q[u][e / 4][e % 4] = qf[gr * 2 + u][e / 4][e % 4];
            }
          }
#pragma unroll
          for (int i = 0; i < NT; ++i) {
            const int row = wslot + i * 8 + (g >> 1) + (g & 1) * 4;  // the slot of column g
            const uint32_t w = *reinterpret_cast<const uint32_t*>(sK + at4<HD, false>(row, gr) + t * 4);
            const uint32_t p0 = *reinterpret_cast<const uint32_t*>(sK + T::kRows + slot_at(i, 0) * T::kPairBytes + gr * 4);
            const uint32_t p1 = *reinterpret_cast<const uint32_t*>(sK + T::kRows + slot_at(i, 1) * T::kPairBytes + gr * 4);
            float c[4] = {0.f, 0.f, 0.f, 0.f};
            const uint32_t n0 = codes_f16(w), n1 = codes16_f16(w), n2 = codes_f16(w >> 8), n3 = codes16_f16(w >> 8);
            if constexpr (!N8) {
              mma_f16(c, q[0][1], n0, n1);
              mma_f16(c, q[1][1], n2, n3);
            }
            mma_f16(c, q[0][0], n0, n1);
            mma_f16(c, q[1][0], n2, n3);
            if constexpr (N8) c[0] += c[2], c[1] += c[3];
            // c is (q . (code - 8)) / back, and the sums of q are divided alike
            const float sc0 = bf16_lo(p0), sc1 = bf16_lo(p1);
            const float mn0 = fmaf(8.f, sc0, bf16_hi(p0)), mn1 = fmaf(8.f, sc1, bf16_hi(p1));
            sh[i][0] = fmaf(c[0], sc0, fmaf(qsum_a[gr], mn0, sh[i][0]));
            sh[i][1] = fmaf(c[1], sc1, fmaf(qsum_a[gr], mn1, sh[i][1]));
            if constexpr (!N8) {
              sh[i][2] = fmaf(c[2], sc0, fmaf(qsum_b[gr], mn0, sh[i][2]));
              sh[i][3] = fmaf(c[3], sc1, fmaf(qsum_b[gr], mn1, sh[i][3]));
            }
          }
        }
#pragma unroll
        for (int i = 0; i < NT; ++i) sh[i][0] *= back_a, sh[i][1] *= back_a, sh[i][2] *= back_b, sh[i][3] *= back_b;
      } else if constexpr (F32) {
        float s0_[NT][4], s1[NT][4], s2[NT][4];  // an accumulator chain per product
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) s0_[i][e] = s1[i][e] = s2[i][e] = 0.f;
#pragma unroll
        for (int ks = 0; ks < HD / 8; ++ks) {
          uint32_t qh[4], ql[4];
#pragma unroll
          for (int e = 0; e < 4; e += N8 ? 2 : 1) {
            const int row = wr * 16 + g + (e & 1) * 8, ch = ks * 2 + (e >> 1);
            split_tf32(*reinterpret_cast<const float*>(sQ + row * HD * 4 + ((ch ^ (row & 7)) << 4) + t * 4), qh[e], ql[e]);
            if constexpr (N8) qh[e + 1] = ql[e];  // a narrow tile: the second terms in rows 8 to 15
          }
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            const int row = wslot + nt * 8 + g;
            uint32_t kh[2], kl[2];
#pragma unroll
            for (int e = 0; e < 2; ++e)
              split_tf32(*reinterpret_cast<const float*>(sK + row * T::kRowBytes + (((ks * 2 + e) ^ (row & 7)) << 4) + t * 4),
                         kh[e], kl[e]);
            mma_tf32(sh[nt], qh, kh[0], kh[1]);
            mma_tf32(s1[nt], qh, kl[0], kl[1]);
            if constexpr (!N8) {
              mma_tf32(s0_[nt], ql, kl[0], kl[1]);
              mma_tf32(s2[nt], ql, kh[0], kh[1]);
            }
          }
        }
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
          for (int e = 0; e < (N8 ? 2 : 4); ++e) {
            if constexpr (N8) sh[i][e] += s1[i][e + 2] + (s1[i][e] + sh[i][e + 2]);
            else sh[i][e] += s0_[i][e] + (s1[i][e] + s2[i][e]);
          }
      } else {
        float ss[NT][4];
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) ss[i][e] = 0.f;
        const int arow = wr * 16 + (lane & 15);
        const uint32_t qa = smem_addr(sQ) + arow * HD * 2;
        const int krow = (lane & 7) + ((lane >> 4) << 3);
#pragma unroll
        for (int ks = 0; ks < HD / 16; ++ks) {
          uint32_t qh[4], qm[4], ql[4];
          const uint32_t at = qa + (((2 * ks + (lane >> 4)) ^ (arow & 7)) << 4);
          ldsm4(qh, at);  // a narrow tile: with the second terms in rows 8 to 15
          ldsm4(ql, at + (N8 ? 1 : 2) * T::kQRows * HD * 2);
          if constexpr (!N8) ldsm4(qm, at + T::kQRows * HD * 2);
#pragma unroll
          for (int np = 0; np < NT / 2; ++np) {
            const int row = wslot + np * 16 + krow;
            uint32_t k4[4];
            ldsm4(k4, smem_addr(sK) + row * T::kRowBytes + (((2 * ks + ((lane >> 3) & 1)) ^ (row & 7)) << 4));
            mma_bf16(sh[2 * np], qh, k4[0], k4[1]);
            mma_bf16(sh[2 * np + 1], qh, k4[2], k4[3]);
            if constexpr (!N8) {
              mma_bf16(ss[2 * np], qm, k4[0], k4[1]);
              mma_bf16(ss[2 * np + 1], qm, k4[2], k4[3]);
            }
            mma_bf16(ss[2 * np], ql, k4[0], k4[1]);
            mma_bf16(ss[2 * np + 1], ql, k4[2], k4[3]);
          }
        }
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
          for (int e = 0; e < (N8 ? 2 : 4); ++e) {
            if constexpr (N8) sh[i][e] += sh[i][e + 2] + ss[i][e];
            else sh[i][e] += ss[i][e];
          }
      }

      // ---- mask: only blocks that some row sees a part of have anything to hide
      const bool edge = k.v.edge(s0, BN, window, sinks);
      if (edge) {
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (!rows_sees(e < 2 ? pa : pb, s0 + slot_at(i, e), window, sinks)) sh[i][e] = kNegInf;
      }

      // ---- online softmax
      float xa = kNegInf, xb = kNegInf;
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        xa = fmaxf(xa, fmaxf(sh[i][0], sh[i][1]));
        if (!N8) xb = fmaxf(xb, fmaxf(sh[i][2], sh[i][3]));
      }
#pragma unroll
      for (int w = 1; w < 4; w <<= 1) {
        xa = fmaxf(xa, __shfl_xor_sync(0xffffffffu, xa, w));
        if (!N8) xb = fmaxf(xb, __shfl_xor_sync(0xffffffffu, xb, w));
      }
      xa = fmaxf(xa, ma), xb = fmaxf(xb, mb);
      // rows that have seen nothing yet keep a maximum of -inf; their p are exp2(-inf - 0) = 0
      const float ba = xa == kNegInf ? 0.f : xa, bb = xb == kNegInf ? 0.f : xb;
      float fa = ex2(ma - ba), fb = N8 ? 1.f : ex2(mb - bb);
      ma = xa, mb = xb;
      float sa = 0.f, sb = 0.f;
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        sh[i][0] = ex2(sh[i][0] - ba), sh[i][1] = ex2(sh[i][1] - ba);
        sa += sh[i][0] + sh[i][1];
        if (N8) continue;
        sh[i][2] = ex2(sh[i][2] - bb), sh[i][3] = ex2(sh[i][3] - bb);
        sb += sh[i][2] + sh[i][3];
      }
      la = la * fa + sa, lb = lb * fb + sb;
      if constexpr (N8) {  // from row g to the rows of o, 2t and 2t + 1
        fb = __shfl_sync(0xffffffffu, fa, 8 * t + 4);
        fa = __shfl_sync(0xffffffffu, fa, 8 * t);
      }

      // ---- o = o * f + p . V, the block's product from a fresh accumulator
      if constexpr (Q4) {
        constexpr int NK = SN / 16;
        const unsigned char* pairs = sV + T::kRows;
        float cm[4] = {0.f, 0.f, 0.f, 0.f};
        uint32_t nan_bits[4] = {0u, 0u, 0u, 0u};
#pragma unroll
        for (int j = 0; j < NK; ++j) {
          // the middles: column g of the product (narrow: row g) is group g; this lane's slots are t, t + 4,
          // t + 8, t + 12
          const int row = wslot + j * 16 + t;
          uint32_t h[4], m[4], l[4];
          float mid[4];
          split3(sh[2 * j][0], sh[2 * j][1], h[0], m[0], l[0]), split3(sh[2 * j + 1][0], sh[2 * j + 1][1], h[2], m[2], l[2]);
          if constexpr (!N8)
            split3(sh[2 * j][2], sh[2 * j][3], h[1], m[1], l[1]), split3(sh[2 * j + 1][2], sh[2 * j + 1][3], h[3], m[3], l[3]);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t pr = *reinterpret_cast<const uint32_t*>(pairs + (row + 4 * e) * T::kPairBytes + (g & (NG - 1)) * 4);
            mid[e] = fmaf(8.f, bf16_lo(pr), bf16_hi(pr));
          }
          if (edge) {
            // A group that was appended with a NaN or an infinity in it has a NaN for its minimum. Where
            // the row is hidden, 0 x NaN must not reach the output: the NaN is taken out, and counted for
            // the rows that see it.
            bool bad = false;
#pragma unroll
            for (int e = 0; e < 4; ++e) bad |= mid[e] != mid[e];
            if (__any_sync(0xffffffffu, bad)) {
              uint32_t seen[4], nan[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                nan[e] = mid[e] != mid[e] ? 0x3f80u : 0u;
                if (nan[e]) mid[e] = 0.f;
                const int p = e & 1 ? pb : pa, at = s0 + row + (e >> 1) * 8;
                seen[e] = (rows_sees(p, at, window, sinks) ? 0x3f80u : 0u) |
                          (rows_sees(p, at + 4, window, sinks) ? 0x3f800000u : 0u);
              }
              float c[4] = {0.f, 0.f, 0.f, 0.f};
              if constexpr (N8) {
                const uint32_t n4[4] = {nan[0] | nan[1] << 16, 0u, nan[2] | nan[3] << 16, 0u};
                mma_bf16(c, n4, seen[0], seen[2]);
              } else {
                mma_bf16(c, seen, nan[0] | nan[1] << 16, nan[2] | nan[3] << 16);
              }
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (c[e] > 0.f) nan_bits[e] = 0x7fc00000u;
            }
          }
          const uint32_t b0 = pack_bf16(mid[0], mid[1]), b1 = pack_bf16(mid[2], mid[3]);
          const uint32_t d0 = pack_bf16(mid[0] - bf16_lo(b0), mid[1] - bf16_hi(b0));
          const uint32_t d1 = pack_bf16(mid[2] - bf16_lo(b1), mid[3] - bf16_hi(b1));
          if constexpr (N8) {
            const uint32_t bd4[4] = {b0, d0, b1, d1};  // rows 8 to 15: the second terms
            mma_bf16(cm, bd4, l[0], l[2]);
            mma_bf16(cm, bd4, m[0], m[2]);
            mma_bf16(cm, bd4, h[0], h[2]);
          } else {
            mma_bf16(cm, l, b0, b1);
            mma_bf16(cm, m, d0, d1);
            mma_bf16(cm, h, d0, d1);
            mma_bf16(cm, m, b0, b1);
            mma_bf16(cm, h, b0, b1);
          }
        }
        if constexpr (N8) cm[0] += cm[2], cm[1] += cm[3];
#pragma unroll
        for (int e = 0; e < (N8 ? 2 : 4); ++e)
          om[e] = nan_bits[e] ? __uint_as_float(nan_bits[e]) : fmaf(om[e], second(e) ? fb : fa, cm[e]);
        // Where rows see only a part of the block, a hidden slot's scale may be far larger than theirs, and with
        // one factor for all it would leave p times theirs few bits, or none. So where the scales of a group are more
        // than 2^10 to 2^17 apart (two fp16 terms lose 2^-25, 2^-22 of what 2^-17 of the largest leaves), each row
        // goes by the scales that it sees (PART). That code is a copy of its own: 64 sequences of 4000 to 8000 slots
        // take 67.8 us with their launches, 66.7 without any of this, 68.6 with the copy for every block that rows
        // see a part of, 71 with these decisions in one loop, 70.7 with the block's slots in turns of like scales.
        auto p_at = [&](int j, int e, int row) { return sh[2 * j + e / 2][e % 2 + 2 * row]; };
        auto scale_at = [&](int j, int e, int gr) {
          return bf16_lo(*reinterpret_cast<const uint32_t*>(pairs + (wslot + j * 16 + t + 4 * e) * T::kPairBytes + gr * 4));
        };
        auto power = [](float m) { return max((int)(__float_as_uint(m) >> 23) | 7, 15); };
        auto most_of_row = [](float m) {
          m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
          return fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
        };
        bool uneven = false;
        if (edge) {
          const uint32_t* own = reinterpret_cast<const uint32_t*>(pairs + (wslot + lane % SN) * T::kPairBytes);  // a lane per slot
#pragma unroll 1
          for (int gr = 0; gr < NG; ++gr) {
            const uint32_t x = own[gr] & 0x7fffu;  // the scale's bits: its exponent from bit 7 on
            const uint32_t most = __reduce_max_sync(0xffffffffu, x) >> 7, least = __reduce_min_sync(0xffffffffu, x ? x : 0x7fffu) >> 7;
            uneven |= least + 17u < (most | 7u);
          }
        }
        auto add_codes = [&](auto part) {
          constexpr bool PART = decltype(part)::value;
#pragma unroll
          for (int gr = 0; gr < NG; ++gr) {
            // Column c of tile i of a group is its dim 8 (c & 3) + 4 (c >> 2) + i: lane (g, t) holds the
            // four nibbles of column g in one half of a word, of two slots side by side in a register. (Narrow:
            // tiles i and i + 1 are the halves of a product's 16 rows.)
            constexpr int NC = N8 ? 2 : 4;
            float c[NC][4];
#pragma unroll
            for (int i = 0; i < NC; ++i)
#pragma unroll
              for (int e = 0; e < 4; ++e) c[i][e] = 0.f;
            float sc[NK][4], most = 0.f;
#pragma unroll
            for (int j = 0; j < NK; ++j)
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                sc[j][e] = scale_at(j, e, gr);
                if constexpr (N8 && PART) sc[j][e] = p_at(j, e, 0) != 0.f ? sc[j][e] : 0.f;
              }
#pragma unroll
            for (int j = 0; j < NK; ++j)
#pragma unroll
              for (int e = 0; e < 4; ++e) most = fmaxf(most, sc[j][e]);
            float most_b = most;
            if constexpr (!N8 && PART) {
              most = most_b = 0.f;
#pragma unroll
              for (int j = 0; j < NK; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  if (p_at(j, e, 0) != 0.f) most = fmaxf(most, sc[j][e]);
                  if (p_at(j, e, 1) != 0.f) most_b = fmaxf(most_b, sc[j][e]);
                }
            }
            most = most_of_row(most);
            if constexpr (!N8 && PART) most_b = most_of_row(most_b);
            else most_b = most;
            // scale * up lies below 2^15; the exponent moves in steps of 8, so that it hardly ever does.
            // (A scale is below 2^109, so both factors are normal numbers.)
            const int ex = power(most), ex_b = N8 ? ex : power(most_b);
            const float up = power_of_two(268 - ex), up_b = power_of_two(268 - ex_b), back = power_of_two(ex - 14);
#pragma unroll
            for (int j = 0; j < NK; ++j) {
              const int row = wslot + j * 16 + t;
              uint32_t w[4], h[4], l[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                w[e] = *reinterpret_cast<const uint16_t*>(sV + at4<HD, true>(row + 4 * e, gr) + (g & 3) * 4 + (g >> 2) * 2);
              }
              float y[4];  // (a scale above the row's own limit is of a hidden slot: cut, so that it times 0 is 0)
#pragma unroll
              for (int e = 0; e < 4; ++e) y[e] = p_at(j, e, 0) * (N8 || !PART ? sc[j][e] * up : fminf(sc[j][e] * up, 0x1p15f));
              split2_f16(y[0], y[1], h[0], l[0]), split2_f16(y[2], y[3], h[2], l[2]);
              if constexpr (!N8) {
#pragma unroll
                for (int e = 0; e < 4; ++e) y[e] = p_at(j, e, 1) * (PART ? fminf(sc[j][e] * up_b, 0x1p15f) : sc[j][e] * up);
                split2_f16(y[0], y[1], h[1], l[1]), split2_f16(y[2], y[3], h[3], l[3]);
              }
              const uint32_t w0 = w[0] | w[1] << 16, w1 = w[2] | w[3] << 16;
#pragma unroll
              for (int i = 0; i < NC; ++i) {
                if constexpr (N8) {
                  const uint32_t u0 = w0 >> (8 * i), u1 = w1 >> (8 * i);
                  const uint32_t v[4] = {codes_f16(u0), codes16_f16(u0), codes_f16(u1), codes16_f16(u1)};
                  mma_f16(c[i], v, l[0], l[2]);
                  mma_f16(c[i], v, h[0], h[2]);
                } else {
                  const uint32_t u0 = w0 >> (i / 2 * 8), u1 = w1 >> (i / 2 * 8);
                  const uint32_t b0 = i % 2 ? codes16_f16(u0) : codes_f16(u0), b1 = i % 2 ? codes16_f16(u1) : codes_f16(u1);
                  mma_f16(c[i], l, b0, b1);
                  mma_f16(c[i], h, b0, b1);
                }
              }
            }
            // o goes by the largest of its rows' units, but by 2^30 at most: what others hold stays far above
            // fp32's smallest number, whatever one row sees.
            float ga = fa, gb = fb;
            if (PART || back != unit[gr]) {
              float top = back, drop_c = back, drop_d = back;
              if constexpr (PART) {
                const float back_b = power_of_two(ex_b - 14);
                top = fmaxf(back, back_b), drop_d = back_b;
#pragma unroll
                for (int w = 4; w < 32; w <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
                if constexpr (N8) {  // from row g to the rows of o
                  drop_c = __shfl_sync(0xffffffffu, back, 8 * t);
                  drop_d = __shfl_sync(0xffffffffu, back, 8 * t + 4);
                }
              }
              const float now = fminf(fmaxf(top, unit[gr]), 0x1p30f), lift = unit[gr] / now;
              drop_c /= now, drop_d /= now;
              ga *= lift, gb *= lift;
              unit[gr] = now;
#pragma unroll
              for (int i = 0; i < NC; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) c[i][e] *= second(e) ? drop_d : drop_c;
            }
#pragma unroll
            for (int i = 0; i < NC; ++i)
#pragma unroll
              for (int e = 0; e < 4; ++e) o[gr * NC + i][e] = fmaf(o[gr * NC + i][e], second(e) ? gb : ga, c[i][e]);
          }
        };
        if (uneven) add_codes(std::true_type{});
        else add_codes(std::false_type{});
      } else {
        // A row of V that some rows do not see may hold infinities or NaN, and 0 x NaN would reach
        // the rows that must not see it: such values are taken out of the tile and added to the
        // rows that do see them.
        if (edge) {
          auto value = [&](int row, int d) -> float {
            const unsigned char* p = sV + row * T::kRowBytes + (((d * (F32 ? 4 : 2) >> 4) ^ (row & 7)) << 4) + (d * (F32 ? 4 : 2) & 15);
            if constexpr (F32) return *reinterpret_cast<const float*>(p);
            else return bf16_to_f32(*reinterpret_cast<const __nv_bfloat16*>(p));
          };
          // (a narrow tile's warps look at their own slots)
          const int from = N8 ? wslot * HD + lane : tid, to = N8 ? (wslot + SN) * HD : BN * HD, step = N8 ? 32 : kThreads;
          int bad = 0;
          for (int i = from; i < to; i += step) bad |= !is_finite(value(i / HD, i % HD));
          if (N8 ? __any_sync(0xffffffffu, bad) : __syncthreads_or(bad)) {
#pragma unroll
            for (int i = 0; i < NO; ++i)
#pragma unroll
              for (int e = 0; e < 4; ++e) o[i][e] *= second(e) ? fb : fa;
            for (int row = wslot; row < wslot + SN; ++row) {
              const bool first = rows_sees(pc, s0 + row, window, sinks), other = rows_sees(pd, s0 + row, window, sinks);
#pragma unroll
              for (int i = 0; i < NO; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  const float v = value(row, dim_at(i, e));
                  if (!is_finite(v) && (second(e) ? other : first)) o[i][e] += v;
                }
            }
            fa = fb = 1.f;
            if (N8) __syncwarp();
            else __syncthreads();
            for (int i = from; i < to; i += step) {
              const int row = i / HD, d = i % HD;
              if (is_finite(value(row, d))) continue;
              unsigned char* p = sV + row * T::kRowBytes + (((d * (F32 ? 4 : 2) >> 4) ^ (row & 7)) << 4) + (d * (F32 ? 4 : 2) & 15);
              if constexpr (F32) *reinterpret_cast<float*>(p) = 0.f;
              else *reinterpret_cast<uint16_t*>(p) = 0;
            }
            if (N8) __syncwarp();
            else __syncthreads();
          }
        }
        if constexpr (F32 && N8) {
          uint32_t ph[NT][2], pl[NT][2];
#pragma unroll
          for (int j = 0; j < NT; ++j)  // slots 2t, 2t + 1 of a group take the places t, t + 4 of the product
            split_tf32_near(sh[j][0], ph[j][0], pl[j][0]), split_tf32_near(sh[j][1], ph[j][1], pl[j][1]);
#pragma unroll
          for (int i = 0; i < NO; ++i) {
            float ch[4] = {0.f, 0.f, 0.f, 0.f}, cs[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int j = 0; j < NT; ++j) {
              uint32_t vh[4], vl[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const int row = wslot + j * 8 + 2 * t + (e >> 1), d = i * 16 + g + (e & 1) * 8;
                split_tf32(*reinterpret_cast<const float*>(sV + row * T::kRowBytes + (((d >> 2) ^ (row & 7)) << 4) + (d & 3) * 4),
                           vh[e], vl[e]);
              }
              mma_tf32(ch, vh, ph[j][0], ph[j][1]);
              mma_tf32(cs, vl, ph[j][0], ph[j][1]);
              mma_tf32(cs, vh, pl[j][0], pl[j][1]);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) o[i][e] = fmaf(o[i][e], e & 1 ? fb : fa, ch[e] + cs[e]);
          }
        } else if constexpr (N8) {
          constexpr int NK = SN / 16;
          uint32_t ph[NK][2], pm[NK][2], pl[NK][2];
#pragma unroll
          for (int j = 0; j < NK; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e) split3(sh[2 * j + e][0], sh[2 * j + e][1], ph[j][e], pm[j][e], pl[j][e]);
          const int vrow = (lane & 7) + ((lane >> 4) << 3);
#pragma unroll
          for (int i = 0; i < NO; ++i) {
            float ch[4] = {0.f, 0.f, 0.f, 0.f}, cs[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int j = 0; j < NK; ++j) {
              const int row = wslot + j * 16 + vrow;
              uint32_t v4[4];
              ldsm4t(v4, smem_addr(sV) + row * T::kRowBytes + (((2 * i + ((lane >> 3) & 1)) ^ (row & 7)) << 4));
              mma_bf16(ch, v4, ph[j][0], ph[j][1]);
              mma_bf16(cs, v4, pm[j][0], pm[j][1]);
              mma_bf16(cs, v4, pl[j][0], pl[j][1]);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) o[i][e] = fmaf(o[i][e], e & 1 ? fb : fa, ch[e] + cs[e]);
          }
        } else if constexpr (F32) {
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
#pragma unroll
            for (int e = 0; e < 4; ++e) o[i][e] = fmaf(o[i][e], e < 2 ? fa : fb, ch[e] + cs[e]);
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
            for (int u = 0; u < 2; ++u)
#pragma unroll
              for (int e = 0; e < 4; ++e) o[2 * np + u][e] = fmaf(o[2 * np + u][e], e < 2 ? fa : fb, ch[u][e] + cs[u][e]);
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

    // ---- results, through shared memory: the slot groups are joined, and rows leave whole
    __syncthreads();  // the ring is free
    constexpr int kPad = T::kPad;
    float* sO = reinterpret_cast<float*>(ring);
    float* sML = sO + WS * RT * kPad;
    if constexpr (N8) {
      float* oc = sO + (ws * RT + 2 * t) * kPad;
      float* od = oc + kPad;
      if constexpr (Q4) {
#pragma unroll
        for (int gr = 0; gr < NG; ++gr) {
          const float m0 = __shfl_sync(0xffffffffu, om[0], gr * 4 + t), m1 = __shfl_sync(0xffffffffu, om[1], gr * 4 + t);
          const int d = gr * kGroup4 + 8 * (g & 3) + 4 * (g >> 2);
          const float(&x)[4] = o[gr * 2];
          const float(&y)[4] = o[gr * 2 + 1];
          const float u = unit[gr], v = u * 0.0625f;
          *reinterpret_cast<float4*>(oc + d) =
              make_float4(fmaf(x[0], u, m0), fmaf(x[2], v, m0), fmaf(y[0], u, m0), fmaf(y[2], v, m0));
          *reinterpret_cast<float4*>(od + d) =
              make_float4(fmaf(x[1], u, m1), fmaf(x[3], v, m1), fmaf(y[1], u, m1), fmaf(y[3], v, m1));
        }
      } else {
#pragma unroll
        for (int i = 0; i < NO; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) (e & 1 ? od : oc)[dim_at(i, e)] = o[i][e];
      }
    } else {
#pragma unroll
      for (int i = 0; i < NO; ++i) {
        float* oa = sO + (ws * RT + ra) * kPad;
        float* ob = sO + (ws * RT + rb) * kPad;
        if constexpr (Q4) {
          const int gr = i / 4, d = gr * kGroup4 + (t & 1) * 16 + (t >> 1) * 4 + i % 4, from = (lane & ~3) | gr >> 1;
          const float m0 = __shfl_sync(0xffffffffu, om[gr & 1], from), m1 = __shfl_sync(0xffffffffu, om[2 + (gr & 1)], from);
          const float u = i % 2 ? unit[gr] * 0.0625f : unit[gr];
          oa[d] = fmaf(o[i][0], u, m0), oa[d + 8] = fmaf(o[i][1], u, m0);
          ob[d] = fmaf(o[i][2], u, m1), ob[d + 8] = fmaf(o[i][3], u, m1);
        } else {
          *reinterpret_cast<float2*>(oa + i * 8 + 2 * t) = make_float2(o[i][0], o[i][1]);
          *reinterpret_cast<float2*>(ob + i * 8 + 2 * t) = make_float2(o[i][2], o[i][3]);
        }
      }
    }
    if (t == 0) {
      sML[(ws * RT + ra) * 2] = ma, sML[(ws * RT + ra) * 2 + 1] = la;
      if (!N8) sML[(ws * RT + rb) * 2] = mb, sML[(ws * RT + rb) * 2 + 1] = lb;
    }
    __syncthreads();
    rows_finish<HD, WS, RT, kThreads>(a, k, b0 == 0 && b1 == k.v.nb, ((size_t)blockIdx.x * 2 + !first_segment) * RT, sO, sML, tid);
    __syncthreads();  // the next segment may use the memory
  });
}

// Joins a tile's segments. W warps share a row: warp w folds the segments w, w + W, ... in order,
// then the warps' results are folded in order, so the sum does not depend on timing. Every
// segment's maximum, sum and output are loaded together: the chain is one load per kBatch segments.
// A warp takes J rows at once: the 36600 rows of two segments that a chunk of 2048 leaves are one
// wave of CTAs with four of them, four waves with one (3 us longer).
template <int HD, int W, int J>
__global__ void __launch_bounds__(kThreads) rows_join_kernel(const __grid_constant__ RowsKernelArgs P, int rt, int bn) {
  constexpr int V = HD / 32, kBatch = J == 1 ? 4 : 2, kRows = 8 / W * J;
  static_assert(J == 1 || W == 1, "shared rows come one at a time");
  __shared__ float so[8][HD], sml[8][2];
  const RowsAttnArgs& a = P.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, w = warp % W;
  const int per = rt / kRows, split = blockIdx.x / per, row0 = blockIdx.x % per * kRows + warp / W * J;
  const RowsTile k(P, P.split_tile[split], rt, bn);
  const int c0 = P.split_cta[split], nsplit = P.split_n[split];
  const int live = k.R - k.r0 - row0;  // rows from row0 on
  // the tile is the first segment of every CTA but the first one, and of that one if it began there
  const bool later = P.begin_tile[c0] != P.split_tile[split];
  launch_next_and_wait();
  float m[J], l[J], acc[J][V];
#pragma unroll
  for (int j = 0; j < J; ++j) {
    m[j] = kNegInf, l[j] = 0.f;
#pragma unroll
    for (int e = 0; e < V; ++e) acc[j][e] = 0.f;
  }
  for (int s0 = w; s0 < nsplit; s0 += kBatch * W) {
    float2 ml[J][kBatch];
    float o[J][kBatch][V];
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const int s = s0 + u * W;
        ml[j][u] = make_float2(kNegInf, 0.f);
#pragma unroll
        for (int e = 0; e < V; ++e) o[j][u][e] = 0.f;
        if (s < nsplit && j < live) {
          const size_t p = ((size_t)(c0 + s) * 2 + (s == 0 && later)) * rt + row0 + j;
          ml[j][u] = *reinterpret_cast<const float2*>(a.part_ml + p * 2);
          if constexpr (V == 4) {
            const float4 f = *reinterpret_cast<const float4*>(a.part_o + p * HD + lane * 4);
            o[j][u][0] = f.x, o[j][u][1] = f.y, o[j][u][2] = f.z, o[j][u][3] = f.w;
          } else {
            const float2 f = *reinterpret_cast<const float2*>(a.part_o + p * HD + lane * 2);
            o[j][u][0] = f.x, o[j][u][1] = f.y;
          }
        }
      }
#pragma unroll
    for (int j = 0; j < J; ++j) {
      float x = m[j];
#pragma unroll
      for (int u = 0; u < kBatch; ++u) x = fmaxf(x, ml[j][u].x);
      const float b = x == kNegInf ? 0.f : x, f = ex2(m[j] - b);
      m[j] = x, l[j] *= f;
#pragma unroll
      for (int e = 0; e < V; ++e) acc[j][e] *= f;
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const float wt = ex2(ml[j][u].x - b);
        l[j] = fmaf(ml[j][u].y, wt, l[j]);
#pragma unroll
        for (int e = 0; e < V; ++e) acc[j][e] = fmaf(o[j][u][e], wt, acc[j][e]);
      }
    }
  }
  if constexpr (W > 1) {
#pragma unroll
    for (int e = 0; e < V; ++e) so[warp][lane * V + e] = acc[0][e];
    if (lane == 0) sml[warp][0] = m[0], sml[warp][1] = l[0];
    __syncthreads();
    if (w != 0) return;
    float x = kNegInf;
#pragma unroll
    for (int u = 0; u < W; ++u) x = fmaxf(x, sml[warp + u][0]);
    const float b = x == kNegInf ? 0.f : x;
    l[0] = 0.f;
#pragma unroll
    for (int e = 0; e < V; ++e) acc[0][e] = 0.f;
#pragma unroll
    for (int u = 0; u < W; ++u) {
      const float wt = ex2(sml[warp + u][0] - b);
      l[0] = fmaf(sml[warp + u][1], wt, l[0]);
#pragma unroll
      for (int e = 0; e < V; ++e) acc[0][e] = fmaf(so[warp + u][lane * V + e], wt, acc[0][e]);
    }
  }
#pragma unroll
  for (int j = 0; j < J; ++j) {
    if (j >= live) return;
    const float inv = 1.0f / l[j];
    float* dst = a.out + ((size_t)k.row0 * a.nq + k.place(k.r0 + row0 + j, a.nq)) * HD + lane * V;
#pragma unroll
    for (int e = 0; e < V; ++e) acc[j][e] *= inv;
    if constexpr (V == 4) *reinterpret_cast<float4*>(dst) = make_float4(acc[j][0], acc[j][1], acc[j][2], acc[j][3]);
    else *reinterpret_cast<float2*>(dst) = make_float2(acc[j][0], acc[j][1]);
  }
}

template <int KIND, int HD, int WR>
cudaError_t configure_one() {
  return cudaFuncSetAttribute(rows_attn_kernel<KIND, HD, WR>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                              Tile<KIND, HD, WR>::kSmem);
}
template <int HD>
cudaError_t configure_hd() {
  cudaError_t e = configure_one<kKvF32, HD, 0>();
  if (e == cudaSuccess) e = configure_one<kKvF32, HD, 1>();
  if (e == cudaSuccess) e = configure_one<kKvF32, HD, 2>();
  if (e == cudaSuccess) e = configure_one<kKvBf16, HD, 0>();
  if (e == cudaSuccess) e = configure_one<kKvBf16, HD, 1>();
  if (e == cudaSuccess) e = configure_one<kKvBf16, HD, 2>();
  if (e == cudaSuccess) e = configure_one<kKv4, HD, 0>();
  if (e == cudaSuccess) e = configure_one<kKv4, HD, 1>();
  if (e == cudaSuccess) e = configure_one<kKv4, HD, 2>();
  return e;
}

template <int KIND, int HD, int WR>
cudaError_t launch(const RowsAttnArgs& a, const RowsBatch& b, int sms, int* launches, cudaStream_t st) {
  using T = Tile<KIND, HD, WR>;
  RowsKernelArgs P;
  const RowsPlan plan = rows_plan(a, b, T::RT, T::BN, sms * T::kCtas, 1, 2, &P);
  const cudaError_t e = launch_early(rows_attn_kernel<KIND, HD, WR>, plan.ctas, kThreads, T::kSmem, st, P);
  *launches += 1;
  return e != cudaSuccess ? e : rows_join(P, plan, T::RT, T::BN, HD, launches, st);
}

// Rows of a sequence that share a KV head, from which on it is a long chunk (rows_attn_tc.cu). Eight
// sequences of 8000 slots, 4 KV heads of 128, with 63 rows and with 70, here against there: bf16 87
// and 134, 139 and 135 us; 4-bit 102 and 141, 171 and 141. An fp32 row costs the tensor cores'
// slow type here: 121 us for 28 rows, 203 against 133 for 35. (One shape: heads of 64, other groups and short
// contexts go by the same numbers, unmeasured.)
bool is_long(const RowsAttnArgs& a, int m, int kind) { return m * (a.nq / a.pages.kvh) > (kind == kKvF32 ? 32 : 64); }

// (KV head, block) pairs of one sequence.
size_t planes_units(const RowsAttnArgs& a, const RowsBatch& b, int i, int kind) {
  return (size_t)a.pages.kvh * RowsView(b.t0[i], b.t0[i] + b.m[i] - 1, a.window, a.sinks, tc_block(kind)).nb;
}
void add(RowsBatch& to, const RowsBatch& b, int i) {
  const int k = to.n_seqs++;
  to.seq[k] = b.seq[i], to.row0[k] = b.row0[i], to.m[k] = b.m[i], to.t0[k] = b.t0[i];
}

template <int KIND, int HD>
cudaError_t launch_short(const RowsAttnArgs& a, const RowsBatch& b, int sms, int* launches, cudaStream_t st) {
  int rows = 0;  // of the largest sequence that share a KV head
  for (int i = 0; i < b.n_seqs; ++i) rows = std::max(rows, b.m[i] * (a.nq / a.pages.kvh));
  // Eight sequences of 8000 slots, 4 KV heads of 128: 7 rows, tiles of 8 against 16 (fp32, bf16, 4-bit):
  // 58, 36, 30 against 82, 40, 42 us; 14 rows, tiles of 16 against 32: 83, 42, 43 against 119,
  // 52, 60. Tiles of 64 gained nothing over two of 32 (63 rows: 87, 102 against 88, 101). One width serves
  // all of a call's short sequences: beside 31 of one row, one of two rows costs 65, 138, 71 us (bf16, fp32,
  // 4-bit; 56, 97, 46 for 32 of one), one of four 87, 208, 105, and in calls of their own 70, 117, 64.
  if (rows <= 8) return launch<KIND, HD, 0>(a, b, sms, launches, st);
  if (rows <= 16) return launch<KIND, HD, 1>(a, b, sms, launches, st);
  return launch<KIND, HD, 2>(a, b, sms, launches, st);
}

// Sequences with few rows in one launch, those with many in another, or in several where their
// fp16 blocks do not fit the scratch together.
template <int KIND, int HD>
cudaError_t launch_kind(const RowsAttnArgs& a, const RowsBatch& b, int sms, int* launches, cudaStream_t st) {
  RowsBatch few;
  few.n_seqs = 0;
  for (int i = 0; i < b.n_seqs; ++i)
    if (!is_long(a, b.m[i], KIND)) add(few, b, i);
  cudaError_t e = few.n_seqs ? launch_short<KIND, HD>(a, few, sms, launches, st) : cudaSuccess;
  RowsBatch many;
  many.n_seqs = 0;
  size_t units = 0;
  for (int i = 0; e == cudaSuccess && i < b.n_seqs; ++i) {
    if (!is_long(a, b.m[i], KIND)) continue;
    const size_t u = planes_units(a, b, i, KIND);
    if (u * tc_unit_bytes(HD) > a.planes_bytes) return cudaErrorInvalidValue;
    if ((units + u) * tc_unit_bytes(HD) > a.planes_bytes) {
      e = launch_rows_tc(a, many, KIND, HD, sms, launches, st);
      many.n_seqs = 0, units = 0;
    }
    add(many, b, i);
    units += u;
  }
  if (e == cudaSuccess && many.n_seqs) e = launch_rows_tc(a, many, KIND, HD, sms, launches, st);
  return e;
}

}  // namespace

RowsPlan rows_plan(const RowsAttnArgs& a, const RowsBatch& b, int rt, int bn, int max_ctas, int least, int start,
                   RowsKernelArgs* P) {
  RowsPlan plan{0, 0, 0, 0};
  P->a = a;
  P->n_seqs = b.n_seqs;
  const int kvh = a.pages.kvh, G = a.nq / kvh;
  std::vector<int> blocks;  // of every tile
  long long total = 0;
  for (int i = 0; i < b.n_seqs; ++i) {
    P->seq[i] = b.seq[i], P->row0[i] = b.row0[i], P->m[i] = b.m[i], P->t0[i] = b.t0[i];
    P->tile0[i] = (int)blocks.size();
    P->unit0[i] = plan.units;
    plan.units += kvh * RowsView(b.t0[i], b.t0[i] + b.m[i] - 1, a.window, a.sinks, bn).nb;
    const int first = (int)blocks.size(), R = b.m[i] * G;
    for (int r0 = 0; r0 < R; r0 += rt)
      blocks.push_back(RowsView(b.t0[i] + r0 / G, b.t0[i] + (std::min(r0 + rt, R) - 1) / G, a.window, a.sinks, bn).nb);
    const int tiles = (int)blocks.size() - first;
    for (int h = 1; h < kvh; ++h)
      for (int t = 0; t < tiles; ++t) blocks.push_back(blocks[first + t]);
    for (size_t t = first; t < blocks.size(); ++t) total += blocks[t];
  }
  const int tiles = (int)blocks.size();
  P->tile0[b.n_seqs] = tiles;
  P->unit0[b.n_seqs] = plan.units;
  max_ctas = std::min(max_ctas, kRowsMaxCtas);
  const int share = std::max((int)((total + max_ctas - 1) / max_ctas), least);
  // the smallest shares with which every tile's blocks are split on their own
  int own = share;
  for (; tiles <= max_ctas && own <= share + start; ++own) {
    int ctas = 0;
    for (int t = 0; t < tiles; ++t) ctas += (blocks[t] + own - 1) / own;
    if (ctas <= max_ctas) break;
  }
  const bool apart = tiles <= max_ctas && own <= share + start;
  int c = 0, left = 0;  // CTAs so far, and what the latest of them may still take
  for (int t = 0; t < tiles; ++t) {
    const int n = (blocks[t] + own - 1) / own;  // apart: the tile's CTAs, as equal as can be
    int first = -1;
    for (int at = 0, k = 0; at < blocks[t]; ++k) {
      if (apart || left == 0) {
        P->begin_tile[c] = t, P->begin_block[c] = at, P->count[c] = 0;
        left = apart ? blocks[t] * (k + 1) / n - at : share;
        ++c;
      }
      const int take = std::min(left, blocks[t] - at);
      P->count[c - 1] += take, left -= take, at += take;
      if (first < 0) first = c - 1;
    }
    if (c - 1 > first) {
      P->split_tile[plan.splits] = t, P->split_cta[plan.splits] = first, P->split_n[plan.splits] = c - first;
      ++plan.splits;
      plan.most_n = std::max(plan.most_n, c - first);
    }
  }
  plan.ctas = c;
  return plan;
}

template <int HD, int W, int J>
cudaError_t launch_join(const RowsKernelArgs& P, int splits, int rt, int bn, cudaStream_t st) {
  return launch_early(rows_join_kernel<HD, W, J>, splits * (rt / (8 / W * J)), kThreads, 0, st, P, rt, bn);
}
template <int HD>
cudaError_t join_hd(const RowsKernelArgs& P, const RowsPlan& plan, int rt, int bn, cudaStream_t st) {
  if (plan.most_n > 8) return launch_join<HD, 8, 1>(P, plan.splits, rt, bn, st);
  return rt % 32 ? launch_join<HD, 1, 1>(P, plan.splits, rt, bn, st) : launch_join<HD, 1, 4>(P, plan.splits, rt, bn, st);
}

cudaError_t rows_join(const RowsKernelArgs& P, const RowsPlan& plan, int rt, int bn, int hd, int* launches, cudaStream_t st) {
  if (plan.splits == 0) return cudaSuccess;
  *launches += 1;
  return hd == 64 ? join_hd<64>(P, plan, rt, bn, st) : join_hd<128>(P, plan, rt, bn, st);
}

// Two partial tiles per CTA, of 256 rows at most with one CTA per SM, and of 8 with two.
size_t rows_attn_part_rows(int sms) { return (size_t)2 * sms * 256; }

size_t rows_attn_planes_bytes(const RowsAttnArgs& a, const RowsBatch& b, int kind, int hd) {
  size_t all = 0, most = 0;
  for (int i = 0; i < b.n_seqs; ++i) {
    if (!is_long(a, b.m[i], kind)) continue;
    const size_t n = planes_units(a, b, i, kind) * tc_unit_bytes(hd);
    all += n, most = std::max(most, n);
  }
  return std::max(most, std::min(all, (size_t)1 << 30));
}

cudaError_t configure_rows_attn() {
  cudaError_t e = configure_hd<64>();
  if (e == cudaSuccess) e = configure_hd<128>();
  if (e == cudaSuccess) e = configure_rows_attn_tc();
  return e;
}

cudaError_t op_rows_attention(const RowsAttnArgs& a, const RowsBatch& b, int kind, int hd, int sms, int* launches,
                              cudaStream_t st) {
  if (!a.part_o || !a.part_ml || !a.err) return cudaErrorInvalidValue;
  switch (kind) {
    case kKvF32:
      return hd == 64 ? launch_kind<kKvF32, 64>(a, b, sms, launches, st) : launch_kind<kKvF32, 128>(a, b, sms, launches, st);
    case kKvBf16:
      return hd == 64 ? launch_kind<kKvBf16, 64>(a, b, sms, launches, st) : launch_kind<kKvBf16, 128>(a, b, sms, launches, st);
    default:
      return hd == 64 ? launch_kind<kKv4, 64>(a, b, sms, launches, st) : launch_kind<kKv4, 128>(a, b, sms, launches, st);
  }
}

}  // namespace dllm
