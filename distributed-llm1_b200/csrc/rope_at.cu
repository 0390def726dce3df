// rope_at.cu — rotary positions per row: q and k of n rows in one launch, each row
// at a position of its own.
//
// For pair i of the first `rotary` dims of a head, (x1, x2) -> (x1 c - x2 s,
// x1 s + x2 c) with c, s = factor * cos, sin(pos * inv_freq[i]); the other dims
// pass. A pair is (i, i + rotary / 2) in the half layout and (2i, 2i + 1) in the
// interleaved one. The angle is reduced in 64 bits: pos * inv_freq / 2 pi is taken
// in turns, whole turns are dropped, and only the remaining half turn goes to
// sincospif in 32 bits. A 32-bit product would be off by pos * 2^-24 radians (0.06 at
// position 10^6). Here the angle is off by two parts: the frequency and its product with
// the position are rounded to 64 bits, about 2^-52 of the whole turns, and what is left of
// a turn to 32, at most pi 2^-25 radians at any position.
//
// Bound by memory (8 bytes per element moved, ~1 flop per byte). A thread owns kVec pairs
// of one head position and keeps their cos and sin in registers while it walks the heads
// of a row, so the trigonometry is done once per row and not once per head. Short rows lie
// side by side in a CTA (6000 rows of 1024 elements, 7.5 us of traffic: 18.6 us with one
// CTA per row, 10.7 so). A CTA ends with its rows: one that stays and loads the next rows
// ahead needs twice the registers and was slower (45.3 against 43.1 us for 8191 rows of
// 4096, whose traffic takes 41.1).
#include "verify.cuh"

namespace dllm {
namespace {

constexpr int kRopeThreads = 256;

template <int VEC>
struct Pack {
  float v[VEC];
};

template <int VEC>
DLLM_DEV Pack<VEC> ld_pack(const float* p) {
  Pack<VEC> r;
  if constexpr (VEC == 4) {
    const float4 f = *reinterpret_cast<const float4*>(p);
    r.v[0] = f.x, r.v[1] = f.y, r.v[2] = f.z, r.v[3] = f.w;
  } else {
    r.v[0] = *p;
  }
  return r;
}
template <int VEC>
DLLM_DEV void st_pack(float* p, const Pack<VEC>& r) {
  if constexpr (VEC == 4)
    *reinterpret_cast<float4*>(p) = make_float4(r.v[0], r.v[1], r.v[2], r.v[3]);
  else
    *p = r.v[0];
}

template <int VEC>
DLLM_DEV Pack<VEC> ld_pack(const __nv_bfloat16* p) {
  Pack<VEC> r;
  if constexpr (VEC == 4) {
    const uint2 f = *reinterpret_cast<const uint2*>(p);
    r.v[0] = bf16_lo(f.x), r.v[1] = bf16_hi(f.x), r.v[2] = bf16_lo(f.y), r.v[3] = bf16_hi(f.y);
  } else {
    r.v[0] = bf16_to_f32(*p);
  }
  return r;
}

// Turns the VEC pairs of a unit.
template <int VEC, bool INTER>
DLLM_DEV void turn(Pack<VEC>& x, Pack<VEC>& y, const float (&c)[VEC], const float (&s)[VEC]) {
  if constexpr (INTER && VEC == 4) {  // (x0 x1)(x2 x3) | (y0 y1)(y2 y3)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float x1 = x.v[2 * i], x2 = x.v[2 * i + 1], y1 = y.v[2 * i], y2 = y.v[2 * i + 1];
      x.v[2 * i] = fmaf(x1, c[i], -(x2 * s[i]));
      x.v[2 * i + 1] = fmaf(x1, s[i], x2 * c[i]);
      y.v[2 * i] = fmaf(y1, c[2 + i], -(y2 * s[2 + i]));
      y.v[2 * i + 1] = fmaf(y1, s[2 + i], y2 * c[2 + i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const float x1 = x.v[i], x2 = y.v[i];
      x.v[i] = fmaf(x1, c[i], -(x2 * s[i]));
      y.v[i] = fmaf(x1, s[i], x2 * c[i]);
    }
  }
}

// A head has hd / (2 VEC) units of VEC pairs: the first rotary / (2 VEC) turn, the
// rest are copied (or left, in place). Four pairs at a time (16-byte accesses)
// need rotary to be a multiple of 8; other sizes go pair by pair, with U heads in flight
// per thread to keep as many bytes under way.
template <int HD, int VEC, int U, bool INTER>
__global__ void __launch_bounds__(kRopeThreads) rope_at_kernel(const RopeAtArgs a, int log2_side) {
  constexpr int units = HD / (2 * VEC), slots = kRopeThreads / units;
  const int turning = a.rotary / (2 * VEC);
  const int heads = a.q_heads + a.k_heads;
  // a CTA's threads: rows, heads side by side (1 << log2_side, the rest in turn), units
  const int unit = threadIdx.x % units, slot = threadIdx.x / units;
  const int h_first = (blockIdx.y << log2_side) + (slot & ((1 << log2_side) - 1)), h_step = gridDim.y << log2_side;
  const int row = blockIdx.x * (slots >> log2_side) + (slot >> log2_side);
  const bool turns = unit < turning;
  // float offsets of the unit's two packs within a head
  const int o1 = turns ? (INTER ? unit * 2 * VEC : unit * VEC) : a.rotary + (unit - turning) * 2 * VEC;
  const int o2 = turns ? (INTER ? o1 + VEC : o1 + a.rotary / 2) : o1 + VEC;
  auto at = [&](int r, int h) {
    return h < a.q_heads ? ((size_t)r * a.q_heads + h) * HD : ((size_t)r * a.k_heads + (h - a.q_heads)) * HD;
  };
  if (row >= a.n) return;
  Pack<VEC> x[U], y[U];
  auto load = [&](int h0) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int h = h0 + u * h_step;
      if (h >= heads) break;
      const float* src = (h < a.q_heads ? a.q : a.k) + at(row, h);
      x[u] = ld_pack<VEC>(src + o1), y[u] = ld_pack<VEC>(src + o2);
    }
  };
  load(h_first);  // on the way while the angles are computed
  float c[VEC], s[VEC];
  if (turns) {
    const double pos = (double)a.pos[row];
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const double t = pos * a.turns[unit * VEC + i];
      sincospif(2.0f * (float)(t - rint(t)), &s[i], &c[i]);
      s[i] *= a.factor;
      c[i] *= a.factor;
    }
  }
  for (int h0 = h_first; h0 < heads; h0 += U * h_step) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int h = h0 + u * h_step;
      if (h >= heads) break;
      if (turns) turn<VEC, INTER>(x[u], y[u], c, s);
      const size_t o = at(row, h);
      float* dst = (h < a.q_heads ? a.q_out : a.k_out) + o;
      if (turns || dst != (h < a.q_heads ? a.q : a.k) + o) {
        st_pack<VEC>(dst + o1, x[u]);
        st_pack<VEC>(dst + o2, y[u]);
      }
    }
    load(h0 + U * h_step);
  }
}

template <int HD, int VEC, int U, bool INTER>
cudaError_t launch_rope(const RopeAtArgs& a, int sms, cudaStream_t st) {
  constexpr int slots = kRopeThreads / (HD / (2 * VEC));
  const int heads = a.q_heads + a.k_heads;
  int log2_side = 0;
  while ((1 << log2_side) < heads && (1 << log2_side) < slots) ++log2_side;
  const int rows = slots >> log2_side, chunks = (heads + (1 << log2_side) - 1) >> log2_side;
  const int ctas = (a.n + rows - 1) / rows;
  // few rows: the heads of a row are spread over CTAs as well, which repeats the
  // angles but leaves one load and store per thread (64 rows of 32 heads: 4.5 us in
  // one CTA per row, 3.3 in two)
  const dim3 grid(ctas, (long long)ctas * chunks <= 8ll * sms ? chunks : 1);
  rope_at_kernel<HD, VEC, U, INTER><<<grid, kRopeThreads, 0, st>>>(a, log2_side);
  return cudaGetLastError();
}

template <int HD>
cudaError_t rope_hd(const RopeAtArgs& a, int sms, cudaStream_t st) {
  if (a.rotary % 8 == 0)
    return a.interleaved ? launch_rope<HD, 4, 1, true>(a, sms, st) : launch_rope<HD, 4, 1, false>(a, sms, st);
  return a.interleaved ? launch_rope<HD, 1, 4, true>(a, sms, st) : launch_rope<HD, 1, 4, false>(a, sms, st);
}

// ---- norms of the heads, then the rotation ---------------------------------------------------
// y = x * rsqrt(mean(x^2) + eps) * w for each head, then the rotation above, in one pass: a
// head's HD / 8 threads (a warp, where pairs go one by one) hold it in registers, add their
// squares in fp32 by shuffles, and turn it. Bound by memory like the rotation alone: the norm
// adds 4 flops per element and one chain of shuffles, and saves a whole pass over q and k.
// 6007 rows of 32 heads of 128: 35 us, 197 MB at 5.6 TB/s (a copy moves 6.6). The next head's
// loads ahead of this one's sum, or the heads of a row over several CTAs, were slower (41, 43):
// more registers and angles taken twice. The weights are loaded before the sum, so that one row
// waits for memory once (7.1 -> 6.3 us; CTAs of 256 threads then cost long batches 2 us).
constexpr int kNormRopeThreads = 128;

template <int HD, int VEC, bool INTER>
__global__ void __launch_bounds__(kNormRopeThreads) norm_rope_kernel(const NormRopeArgs n, int log2_side) {
  constexpr int units = HD / (2 * VEC), lanes = units < 32 ? units : 32, U = units / lanes, slots = kNormRopeThreads / lanes;
  const RopeAtArgs& a = n.rope;
  const int turning = a.rotary / (2 * VEC), heads = a.q_heads + a.k_heads;
  const int lane = threadIdx.x % lanes, slot = threadIdx.x / lanes;
  const int h_first = (blockIdx.y << log2_side) + (slot & ((1 << log2_side) - 1)), h_step = gridDim.y << log2_side;
  const int row = blockIdx.x * (slots >> log2_side) + (slot >> log2_side);
  if (row >= a.n) return;  // a head's threads leave together
  launch_next_and_wait();
  const unsigned group = (lanes == 32 ? 0xffffffffu : (1u << (lanes & 31)) - 1) << (threadIdx.x % 32 - lane);
  // float offsets of this thread's packs within a head
  int o1[U], o2[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int unit = lane + u * lanes;
    const bool turns = unit < turning;
    o1[u] = turns ? (INTER ? unit * 2 * VEC : unit * VEC) : a.rotary + (unit - turning) * 2 * VEC;
    o2[u] = turns ? (INTER ? o1[u] + VEC : o1[u] + a.rotary / 2) : o1[u] + VEC;
  }
  auto at = [&](int h) {
    return h < a.q_heads ? ((size_t)row * a.q_heads + h) * HD : ((size_t)row * a.k_heads + (h - a.q_heads)) * HD;
  };
  Pack<VEC> x[U], y[U];
  auto load = [&](int h) {
    if (h >= heads) return;
    const float* src = (h < a.q_heads ? a.q : a.k) + at(h);
#pragma unroll
    for (int u = 0; u < U; ++u) x[u] = ld_pack<VEC>(src + o1[u]), y[u] = ld_pack<VEC>(src + o2[u]);
  };
  load(h_first);  // on the way while the angles are computed
  float c[U][VEC], s[U][VEC];
  const double pos = (double)a.pos[row];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (lane + u * lanes >= turning) continue;
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const double t = pos * a.turns[(lane + u * lanes) * VEC + i];
      sincospif(2.0f * (float)(t - rint(t)), &s[u][i], &c[u][i]);
      s[u][i] *= a.factor;
      c[u][i] *= a.factor;
    }
  }
  for (int h = h_first; h < heads; h += h_step) {
    const __nv_bfloat16* w = h < a.q_heads ? n.q_norm : n.k_norm;  // from L1 but for the first head
    Pack<VEC> wx[U], wy[U];
#pragma unroll
    for (int u = 0; u < U; ++u) wx[u] = ld_pack<VEC>(w + o1[u]), wy[u] = ld_pack<VEC>(w + o2[u]);
    float sum = 0.f;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < VEC; ++i) sum = fmaf(x[u].v[i], x[u].v[i], fmaf(y[u].v[i], y[u].v[i], sum));
#pragma unroll
    for (int d = lanes / 2; d > 0; d >>= 1) sum += __shfl_xor_sync(group, sum, d);
    const float r = rsqrtf(fmaf(sum, 1.f / HD, n.eps));
    float* dst = (h < a.q_heads ? a.q_out : a.k_out) + at(h);
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        x[u].v[i] *= r * wx[u].v[i];
        y[u].v[i] *= r * wy[u].v[i];
      }
      if (lane + u * lanes < turning) turn<VEC, INTER>(x[u], y[u], c[u], s[u]);
      st_pack<VEC>(dst + o1[u], x[u]);
      st_pack<VEC>(dst + o2[u], y[u]);
    }
    load(h + h_step);
  }
}

template <int HD, int VEC, bool INTER>
cudaError_t launch_norm_rope(const NormRopeArgs& n, int sms, cudaStream_t st) {
  constexpr int units = HD / (2 * VEC), slots = kNormRopeThreads / (units < 32 ? units : 32);
  const RopeAtArgs& a = n.rope;
  const int heads = a.q_heads + a.k_heads;
  int log2_side = 0;
  while ((1 << log2_side) < heads && (1 << log2_side) < slots) ++log2_side;
  const int rows = slots >> log2_side, chunks = (heads + (1 << log2_side) - 1) >> log2_side;
  const int ctas = (a.n + rows - 1) / rows;
  const dim3 grid(ctas, (long long)ctas * chunks <= 8ll * sms ? chunks : 1);  // as above
  return launch_early(norm_rope_kernel<HD, VEC, INTER>, grid, kNormRopeThreads, 0, st, n, log2_side);
}

template <int HD>
cudaError_t norm_rope_hd(const NormRopeArgs& n, int sms, cudaStream_t st) {
  if (n.rope.rotary % 8 == 0)
    return n.rope.interleaved ? launch_norm_rope<HD, 4, true>(n, sms, st) : launch_norm_rope<HD, 4, false>(n, sms, st);
  return n.rope.interleaved ? launch_norm_rope<HD, 1, true>(n, sms, st) : launch_norm_rope<HD, 1, false>(n, sms, st);
}

}  // namespace

cudaError_t op_rope_at(const RopeAtArgs& a, int sms, cudaStream_t st) {
  return a.hd == 64 ? rope_hd<64>(a, sms, st) : rope_hd<128>(a, sms, st);
}

cudaError_t op_norm_rope(const NormRopeArgs& n, int sms, cudaStream_t st) {
  return n.rope.hd == 64 ? norm_rope_hd<64>(n, sms, st) : norm_rope_hd<128>(n, sms, st);
}

}  // namespace dllm
