// kv4.cu — rows of a batch into a paged cache (fp32, bf16 or 4-bit), and 4-bit rows back.
//
// 4 bits: every 32 dims of a head's row share a scale s and a minimum m, both bf16, and each
// value x becomes a code c of 0..15 that stands for m + c s:
//   m = the group's smallest value, rounded down;  s = (largest - m) / 15, rounded up;
//   c = (x - m) / s to the nearest whole number, ties to even
// (x - m, largest - m and the quotients are rounded to fp32). Rounding m down and s up keeps
// every value inside [m, m + 15 s], so each is off by at most s / 2 (and the fp32 rounding).
// A group with a NaN, a number beyond the largest bf16 one (3.39e38: no m below it, or no middle near
// it), an infinity among them, or a range of 2^112 or more (no scale that kernels multiply freely) has
// m = NaN: all its values read NaN.
//
// Memory-bound: 4 bytes in and 5 bits out per value. A thread takes 8 dims of K and of V (four
// 16-byte loads under way, one word of codes each); the four threads of a group exchange
// their extremes in two shuffles. 8185 rows of 4 KV heads of 128: stored and read back in 17.1
// us, 77 MB at 4.5 TB/s (a copy moves 6.6): two launches of 9 us, of which each spends 3 on
// one chain of page table, loads and stores. Sixteen dims per thread were slower (31.7 against 27.6
// us for the pair, before the sectors below were filled).

#include "rows_attn.cuh"

namespace dllm {
namespace {

constexpr int kThreads = 256;

constexpr float kBf16Most = 0x1.fep127f;
DLLM_DEV float bf16_down(float x) {  // the largest bf16 that is not above x (|x| <= kBf16Most)
  uint32_t u = __float_as_uint(x);
  if (x < 0.f) u += 0xffffu;
  return __uint_as_float(u & 0xffff0000u);
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
  for (int e = 0; e < 8; ++e) lo = fminf(lo, x[e]), hi = fmaxf(hi, x[e]), fine = fine && fabsf(x[e]) <= kBf16Most;
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
  // A product with 1 / s is within 2^-19 of the quotient, so both round to one code unless the
  // product is that close to a half (or 1 / s is infinite): only then the quotient is taken.
  const float inv = 1.f / s;
  uint32_t codes = 0;
  bool sure = true;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float t = (x[e] - m) * inv, r = rintf(t);
    sure = sure && fabsf(t - r) < 0.4999f;
    codes |= (uint32_t)__float2int_rn(r) << (4 * e);
  }
  if (sure) return codes;
  codes = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) codes |= (uint32_t)min(__float2int_rn((x[e] - m) / s), 15) << (4 * e);
  return codes;
}

// Thread `at` takes 8 dims: 4 from dim 4 j on, 4 from dim 16 + 4 j on, of group at / 4, j = at % 4.
// Four lanes fill two whole sectors of fp32 then, not four halves (the same 8185 rows: 27.6 us
// with 8 dims in a row per thread, 23.5 so, launches included).
template <int HD>
DLLM_DEV size_t cache_row(const RowsBatch& b, const RowPages& p, unsigned at) {
  const unsigned rh = at / (HD / 8), row = rh / (unsigned)p.kvh;
  const int q = find_seq(b, (int)row);
  return p.row(b.seq[q], b.t0[q] + (int)row - b.row0[q], (int)(rh - row * (unsigned)p.kvh));
}
DLLM_DEV size_t first4(unsigned at) { return (size_t)(at / 4) * 8 + at % 4; }  // the thread's first 4 dims; the others: + 4
// Of the group's four words of codes, the one that lane j stores or loads: even lanes take the words
// of the first 16 dims, odd ones those of the others, and two neighbours exchange a half.
DLLM_DEV unsigned word_of(unsigned j) { return (j & 1) * 2 + j / 2; }

template <int KIND, int HD>
__global__ void __launch_bounds__(kThreads)
    rows_append_kernel(const __grid_constant__ RowsBatch b, unsigned total, RowPages p, const float* k, const float* v,
                       void* kc, void* vc, uint32_t* ks, uint32_t* vs) {
  constexpr int C = HD / 8;
  launch_next_and_wait();
  const unsigned i = blockIdx.x * kThreads + threadIdx.x, at = min(i, total - 1);  // whole warps take part in the shuffles
  const size_t src = first4(at);
  const float4 *k4 = reinterpret_cast<const float4*>(k) + src, *v4 = reinterpret_cast<const float4*>(v) + src;
  const float4 f[4] = {__ldcs(k4), __ldcs(k4 + 4), __ldcs(v4), __ldcs(v4 + 4)};
  const size_t dst = cache_row<HD>(b, p, at);
  const unsigned j = at % 4, group = at % C / 4;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    const float4 g = f[2 * which], h = f[2 * which + 1];
    if constexpr (KIND == kKv4) {
      const float x[8] = {g.x, g.y, g.z, g.w, h.x, h.y, h.z, h.w};
      uint32_t pair;
      const uint32_t codes = encode(x, pair);  // low half: dims 4 j, high half: 16 + 4 j
      const uint32_t other = __shfl_xor_sync(0xffffffffu, codes, 1);
      const uint32_t word = j & 1 ? __byte_perm(other, codes, 0x7632) : __byte_perm(codes, other, 0x5410);
      if (i >= total) continue;
      static_cast<uint32_t*>(which ? vc : kc)[dst * C + group * 4 + word_of(j)] = word;
      if (j == 0) (which ? vs : ks)[dst * (C / 4) + group] = pair;
    } else {
      if (i >= total) continue;
      const size_t o = dst * (HD / 4) + group * 8 + j;
      if constexpr (KIND == kKvF32) {
        float4* out = static_cast<float4*>(which ? vc : kc) + o;
        out[0] = g, out[4] = h;
      } else {  // the cache's own rounding: to nearest, ties to even
        uint2* out = static_cast<uint2*>(which ? vc : kc) + o;
        out[0] = make_uint2(pack_bf16(g.x, g.y), pack_bf16(g.z, g.w));
        out[4] = make_uint2(pack_bf16(h.x, h.y), pack_bf16(h.z, h.w));
      }
    }
  }
}

template <int HD>
__global__ void __launch_bounds__(kThreads)
    rows_read4_kernel(const __grid_constant__ RowsBatch b, unsigned total, RowPages p, const uint32_t* kc,
                      const uint32_t* vc, const uint32_t* ks, const uint32_t* vs, float* k, float* v) {
  constexpr int C = HD / 8;
  launch_next_and_wait();
  const unsigned i = blockIdx.x * kThreads + threadIdx.x, at = min(i, total - 1);
  const size_t src = cache_row<HD>(b, p, at), dst = first4(at);
  const unsigned j = at % 4, group = at % C / 4;
  uint32_t word[2] = {0u, 0u}, pair[2] = {0u, 0u};
  if (k) word[0] = kc[src * C + group * 4 + word_of(j)], pair[0] = ks[src * (C / 4) + group];
  if (v) word[1] = vc[src * C + group * 4 + word_of(j)], pair[1] = vs[src * (C / 4) + group];
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    const uint32_t other = __shfl_xor_sync(0xffffffffu, word[which], 1);
    float4* out = reinterpret_cast<float4*>(which ? v : k);
    if (!out || i >= total) continue;
    const uint32_t codes = j & 1 ? __byte_perm(other, word[which], 0x7632) : __byte_perm(word[which], other, 0x5410);
    const float s = bf16_lo(pair[which]), m = bf16_hi(pair[which]);
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = fmaf((float)(codes >> (4 * e) & 15u), s, m);
    out[dst] = make_float4(x[0], x[1], x[2], x[3]);
    out[dst + 4] = make_float4(x[4], x[5], x[6], x[7]);
  }
}

unsigned units_of(int n, int kvh, int hd) { return (unsigned)n * kvh * (hd / 8); }
unsigned grid_of(unsigned units) { return (units - 1) / kThreads + 1; }

template <int KIND>
cudaError_t append(const RowsBatch& b, int n, const RowPages& p, int hd, const float* k, const float* v, void* kc, void* vc,
                   uint32_t* ks, uint32_t* vs, cudaStream_t st) {
  const unsigned units = units_of(n, p.kvh, hd), grid = grid_of(units);
  const auto kernel = hd == 64 ? rows_append_kernel<KIND, 64> : rows_append_kernel<KIND, 128>;
  return launch_early(kernel, grid, kThreads, 0, st, b, units, p, k, v, kc, vc, ks, vs);
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
  const unsigned units = units_of(n, p.kvh, hd), grid = grid_of(units);
  const uint32_t *kw = static_cast<const uint32_t*>(kc), *vw = static_cast<const uint32_t*>(vc);
  const auto kernel = hd == 64 ? rows_read4_kernel<64> : rows_read4_kernel<128>;
  return launch_early(kernel, grid, kThreads, 0, st, b, units, p, kw, vw, ks, vs, k, v);
}

}  // namespace dllm
