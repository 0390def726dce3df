// kv4.cu — rows of a batch into a paged cache (fp32, bf16 or 4-bit), and 4-bit rows back.
//
// 4 bits: every 32 dims of a head's row share a scale s and a minimum m, both bf16, and each
// value x becomes a code c of 0..15 that stands for m + c s:
//   m = the group's smallest value, rounded down;  s = (largest - m) / 15, rounded up;
//   c = (x - m) / s to the nearest whole number, ties to even
// (x - m, largest - m and the quotients are rounded to fp32). Rounding m down and s up keeps
// every value inside [m, m + 15 s], so each is off by at most s / 2 (and the fp32 rounding).
// A group with a NaN, an infinity, or a range of 2^112 or more (no scale that kernels multiply
// freely) has m = NaN: all its values read NaN.
//
// Memory-bound: 4 bytes in and 5 bits out per value. A thread takes 8 dims of K and of V (four
// 16-byte loads under way, one word of codes each); the four threads of a group exchange
// their extremes in two shuffles.

#include "rows_attn.cuh"

namespace dllm {
namespace {

constexpr int kThreads = 256;

DLLM_DEV float bf16_down(float x) {  // the largest finite bf16 that is not above x (x finite)
  uint32_t u = __float_as_uint(x);
  if (x < 0.f) u += 0xffffu;
  u &= 0xffff0000u;
  return __uint_as_float(u == 0xff800000u ? 0xff7f0000u : u);
}
DLLM_DEV float bf16_up(float x) {  // the smallest bf16 that is not below x (x >= 0, far from the largest)
  return __uint_as_float((__float_as_uint(x) + 0xffffu) & 0xffff0000u);
}
DLLM_DEV int find_seq(const RowsBatch& b, int row) {
  int lo = 0, hi = b.n_seqs;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (b.row0[mid] <= row) lo = mid;
    else hi = mid;
  }
  return lo;
}

// The codes of 8 values of a group; every lane of the group's four returns the pair. All 32
// lanes call it.
DLLM_DEV uint32_t encode(const float (&x)[8], uint32_t& pair) {
  float lo = x[0], hi = x[0];
  bool fine = true;
#pragma unroll
  for (int e = 0; e < 8; ++e) lo = fminf(lo, x[e]), hi = fmaxf(hi, x[e]), fine = fine && is_finite(x[e]);
#pragma unroll
  for (int w = 1; w < 4; w <<= 1) {
    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, w));
    hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, w));
    fine = __shfl_xor_sync(0xffffffffu, (int)fine, w) && fine;
  }
  const float m = bf16_down(lo), range = hi - m;
  if (!fine || !(range < 0x1p112f)) {
    pair = 0x7fc00000u;
    return 0u;
  }
  const float s = bf16_up(range / 15.f);
  pair = __float_as_uint(s) >> 16 | (__float_as_uint(m) & 0xffff0000u);
  if (s == 0.f) return 0u;
  uint32_t codes = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) codes |= (uint32_t)min(__float2int_rn((x[e] - m) / s), 15) << (4 * e);
  return codes;
}

template <int KIND, int HD>
__global__ void __launch_bounds__(kThreads)
    rows_append_kernel(const __grid_constant__ RowsBatch b, int n, RowPages p, const float* k, const float* v, void* kc,
                       void* vc, uint32_t* ks, uint32_t* vs) {
  constexpr int C = HD / 8;
  const int kvh = p.kvh;
  const long long total = (long long)n * kvh * C, i = (long long)blockIdx.x * kThreads + threadIdx.x;
  const long long at = min(i, total - 1);  // whole warps take part in the shuffles
  const int c = (int)(at % C);
  const long long rh = at / C;
  const int row = (int)(rh / kvh), head = (int)(rh % kvh);
  const float4 *ksrc = reinterpret_cast<const float4*>(k + at * 8), *vsrc = reinterpret_cast<const float4*>(v + at * 8);
  const float4 f[4] = {ksrc[0], ksrc[1], vsrc[0], vsrc[1]};
  const int q = find_seq(b, row);
  const size_t dst = p.row(b.seq[q], b.t0[q] + row - b.row0[q], head);
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    const float4 g = f[2 * which], h = f[2 * which + 1];
    if constexpr (KIND == kKv4) {
      const float x[8] = {g.x, g.y, g.z, g.w, h.x, h.y, h.z, h.w};
      uint32_t pair;
      const uint32_t codes = encode(x, pair);
      if (i >= total) continue;
      static_cast<uint32_t*>(which ? vc : kc)[dst * C + c] = codes;
      if (c % 4 == 0) (which ? vs : ks)[dst * (C / 4) + c / 4] = pair;
    } else {
      if (i >= total) continue;
      if constexpr (KIND == kKvF32) {
        float4* out = static_cast<float4*>(which ? vc : kc) + dst * (HD / 4) + c * 2;
        out[0] = g, out[1] = h;
      } else {  // the cache's own rounding: to nearest, ties to even
        static_cast<uint4*>(which ? vc : kc)[dst * C + c] =
            make_uint4(pack_bf16(g.x, g.y), pack_bf16(g.z, g.w), pack_bf16(h.x, h.y), pack_bf16(h.z, h.w));
      }
    }
  }
}

template <int HD>
__global__ void __launch_bounds__(kThreads)
    rows_read4_kernel(const __grid_constant__ RowsBatch b, int n, RowPages p, const uint32_t* kc, const uint32_t* vc,
                      const uint32_t* ks, const uint32_t* vs, float* k, float* v) {
  constexpr int C = HD / 8;
  const long long total = (long long)n * p.kvh * C, at = (long long)blockIdx.x * kThreads + threadIdx.x;
  if (at >= total) return;
  const int c = (int)(at % C);
  const long long rh = at / C;
  const int row = (int)(rh / p.kvh), head = (int)(rh % p.kvh);
  const int q = find_seq(b, row);
  const size_t src = p.row(b.seq[q], b.t0[q] + row - b.row0[q], head);
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    float* out = which ? v : k;
    if (!out) continue;
    const uint32_t codes = (which ? vc : kc)[src * C + c], pair = (which ? vs : ks)[src * (C / 4) + c / 4];
    const float s = bf16_lo(pair), m = bf16_hi(pair);
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = fmaf((float)(codes >> (4 * e) & 15u), s, m);
    reinterpret_cast<float4*>(out + at * 8)[0] = make_float4(x[0], x[1], x[2], x[3]);
    reinterpret_cast<float4*>(out + at * 8)[1] = make_float4(x[4], x[5], x[6], x[7]);
  }
}

unsigned grid_of(int n, int kvh, int hd) { return (unsigned)(((long long)n * kvh * (hd / 8) + kThreads - 1) / kThreads); }

template <int KIND>
cudaError_t append(const RowsBatch& b, int n, const RowPages& p, int hd, const float* k, const float* v, void* kc, void* vc,
                   uint32_t* ks, uint32_t* vs, cudaStream_t st) {
  const unsigned grid = grid_of(n, p.kvh, hd);
  if (hd == 64) rows_append_kernel<KIND, 64><<<grid, kThreads, 0, st>>>(b, n, p, k, v, kc, vc, ks, vs);
  else rows_append_kernel<KIND, 128><<<grid, kThreads, 0, st>>>(b, n, p, k, v, kc, vc, ks, vs);
  return cudaGetLastError();
}

}  // namespace

cudaError_t op_rows_append(const RowsBatch& b, int n, const RowPages& p, int kind, int hd, const float* k, const float* v,
                           void* kc, void* vc, uint32_t* ks, uint32_t* vs, cudaStream_t st) {
  if (kind == kKvF32) return append<kKvF32>(b, n, p, hd, k, v, kc, vc, ks, vs, st);
  if (kind == kKvBf16) return append<kKvBf16>(b, n, p, hd, k, v, kc, vc, ks, vs, st);
  return append<kKv4>(b, n, p, hd, k, v, kc, vc, ks, vs, st);
}

cudaError_t op_rows_read4(const RowsBatch& b, int n, const RowPages& p, int hd, const void* kc, const void* vc,
                          const uint32_t* ks, const uint32_t* vs, float* k, float* v, cudaStream_t st) {
  const unsigned grid = grid_of(n, p.kvh, hd);
  const uint32_t *kw = static_cast<const uint32_t*>(kc), *vw = static_cast<const uint32_t*>(vc);
  if (hd == 64) rows_read4_kernel<64><<<grid, kThreads, 0, st>>>(b, n, p, kw, vw, ks, vs, k, v);
  else rows_read4_kernel<128><<<grid, kThreads, 0, st>>>(b, n, p, kw, vw, ks, vs, k, v);
  return cudaGetLastError();
}

}  // namespace dllm
