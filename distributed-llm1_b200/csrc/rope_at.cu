// rope_at.cu — rotary positions per row: q and k of n rows in one launch, each row
// at a position of its own.
//
// For pair i of the first `rotary` dims of a head, (x1, x2) -> (x1 c - x2 s,
// x1 s + x2 c) with c, s = factor * cos, sin(pos * inv_freq[i]); the other dims
// pass. A pair is (i, i + rotary / 2) in the half layout and (2i, 2i + 1) in the
// interleaved one. The angle is reduced in 64 bits: pos * inv_freq / 2 pi is taken
// in turns, whole turns are dropped, and only the remaining half turn goes to
// sincospif in 32 bits. A 32-bit product would be off by pos * 2^-24 radians
// (0.06 at position 10^6); this form stays within 2^-52 * turns of the angle.
//
// Bound by memory (8 bytes per element moved, ~1 flop per byte). A thread owns
// kVec pairs of one head position and keeps their cos and sin in registers while
// it walks the heads of the row, so the trigonometry is done once per row and not
// once per head.
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

// A head has hd / (2 VEC) units of VEC pairs: the first rotary / (2 VEC) turn, the
// rest are copied (or left, in place). Four pairs at a time (16-byte accesses)
// need rotary to be a multiple of 8; other sizes go pair by pair.
template <int VEC, bool INTER>
__global__ void __launch_bounds__(kRopeThreads) rope_at_kernel(const RopeAtArgs a) {
  const int units = a.hd / (2 * VEC);
  const int turning = a.rotary / (2 * VEC);
  const int unit = threadIdx.x % units;
  const int per = kRopeThreads / units;  // heads in flight
  const int heads = a.q_heads + a.k_heads;
  const int row = blockIdx.x;
  const bool turns = unit < turning;
  // float offsets of the unit's two packs within a head
  const int o1 = turns ? (INTER ? unit * 2 * VEC : unit * VEC) : a.rotary + (unit - turning) * 2 * VEC;
  const int o2 = turns ? (INTER ? o1 + VEC : o1 + a.rotary / 2) : o1 + VEC;
  // the first head's elements are on their way while the angles are computed
  auto head_at = [&](int h, const float*& src, float*& dst) {
    const bool is_q = h < a.q_heads;
    const size_t at = is_q ? ((size_t)row * a.q_heads + h) * a.hd : ((size_t)row * a.k_heads + (h - a.q_heads)) * a.hd;
    src = (is_q ? a.q : a.k) + at;
    dst = (is_q ? a.q_out : a.k_out) + at;
  };
  const float* src;
  float* dst;
  int h = blockIdx.y * per + threadIdx.x / units;
  Pack<VEC> x, y;
  if (h < heads) {
    head_at(h, src, dst);
    x = ld_pack<VEC>(src + o1), y = ld_pack<VEC>(src + o2);
  }
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
  while (h < heads) {
    if (turns) {
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
    if (turns || src != dst) {
      st_pack<VEC>(dst + o1, x);
      st_pack<VEC>(dst + o2, y);
    }
    h += per * gridDim.y;
    if (h < heads) {
      head_at(h, src, dst);
      x = ld_pack<VEC>(src + o1), y = ld_pack<VEC>(src + o2);
    }
  }
}

}  // namespace

cudaError_t op_rope_at(const RopeAtArgs& a, int sms, cudaStream_t st) {
  const bool vec = a.rotary % 8 == 0;
  // few rows: the heads of a row are spread over CTAs as well, which repeats the
  // angles but leaves one load and store per thread (64 rows of 32 heads: 4.5 us in
  // one CTA per row)
  const int per = kRopeThreads / (a.hd / (vec ? 8 : 2));
  const int chunks = (a.q_heads + a.k_heads + per - 1) / per;
  const dim3 grid(a.n, (long long)a.n * chunks <= 8ll * sms ? chunks : 1);
  if (vec && a.interleaved)
    rope_at_kernel<4, true><<<grid, kRopeThreads, 0, st>>>(a);
  else if (vec)
    rope_at_kernel<4, false><<<grid, kRopeThreads, 0, st>>>(a);
  else if (a.interleaved)
    rope_at_kernel<1, true><<<grid, kRopeThreads, 0, st>>>(a);
  else
    rope_at_kernel<1, false><<<grid, kRopeThreads, 0, st>>>(a);
  return cudaGetLastError();
}

}  // namespace dllm
