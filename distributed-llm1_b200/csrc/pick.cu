// pick.cu — one token per row of logits under penalties for repeated tokens,
// additive biases and a grammar mask, and the processed logits where they are wanted.
//
// For token t of a row with logit x, c = occurrences among the generated tokens:
//   y = x > 0 ? x / repetition : x * repetition     if t occurs in the history at all
//   y = (y - frequency * c) - presence              if c > 0
//   y = y + bias[t]                                 if t is in the bias list
//   y = -inf                                        if the mask forbids t
// and the pick is the first allowed t with the largest y (NaN counts as -inf), -1
// where the mask allows nothing. Every step is one rounded 32-bit operation, as
// separate elementwise operations would round it. The history of a tree's node is
// its sequence's tokens, then the drafted tokens on the path from the root to it.
//
// Bound by memory: the logits are read once (and written once); history, biases
// and mask are small beside them. A CTA takes one slice of the vocabulary for one
// row, or for several nodes of a tree: it counts the history's tokens that fall into
// its slice in shared memory (integer atomics, so their order does not matter) and
// streams its slice of those rows, a tree's node correcting the counts by the path
// tokens it does not share with the node before. A thread keeps U 16-byte groups of
// a row in registers and loads the next row's as it uses them up, the first row's
// before the counting, so the logits stay in flight throughout. The slices' best
// (value, index) keys meet in one 64-bit atomicMax per row (the largest key wins in
// any order); the CTA that arrives last writes the token and clears the key.
#include <algorithm>
#include <climits>

#include "verify.cuh"

namespace dllm {
namespace {

constexpr int kPickThreads = 512;
constexpr int kPickWarps = kPickThreads / 32;
constexpr int kMaxRowsPerCta = 16;

constexpr uint32_t kGiven = 0x80000000u;  // the token occurs among the given (prompt) tokens

// Best allowed token so far of one thread, which sees tokens in ascending order.
struct Best {
  float v = -INFINITY;
  int t = -1;
  DLLM_DEV void see(float y, int tok) {
    if (t < 0 || y > v) {  // a NaN is never greater
      v = y == y ? y : -INFINITY;
      t = tok;
    }
  }
};

struct RowRules {
  float rep, freq, pres;
  const float* bias_val;  // the sequence's bias entries
};

// The rules above for one token. cnt: its count word; b: 1 + its entry in the bias
// list, or 0.
DLLM_DEV float apply(float x, uint32_t cnt, uint32_t b, const RowRules& r) {
  if (cnt) {
    x = x > 0.f ? __fdiv_rn(x, r.rep) : __fmul_rn(x, r.rep);
    const uint32_t c = cnt & ~kGiven;
    if (c) x = __fsub_rn(__fsub_rn(x, __fmul_rn(r.freq, (float)c)), r.pres);
  }
  if (b) x = __fadd_rn(x, r.bias_val[b - 1]);
  return x;
}

DLLM_DEV int clampi(int v, int lo, int hi) { return v < lo ? lo : (v > hi ? hi : v); }

// One 16-byte group of a row: tokens [t, t + 4), some of which may lie outside the
// vocabulary at a row's ends (rows whose length is no multiple of 4 start inside a
// group). bits: which of the four are allowed tokens.
struct Group {
  float v[4];
  uint32_t bits;
};

DLLM_DEV void load_group(Group& g, const float* x, const uint32_t* mask, int t, int vocab) {
  if (t >= 0 && t + 3 < vocab) {
    const float4 f = __ldcs(reinterpret_cast<const float4*>(x + t));
    g.v[0] = f.x, g.v[1] = f.y, g.v[2] = f.z, g.v[3] = f.w;
    g.bits = 0xfu;
    if (mask) {
      const int w = t >> 5, sh = t & 31;
      g.bits = mask[w] >> sh;
      if (sh > 28) g.bits |= mask[w + 1] << (32 - sh);
    }
  } else {
    g.bits = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int tok = t + e;
      g.v[e] = 0.f;
      if (tok < 0 || tok >= vocab) continue;
      g.v[e] = x[tok];
      if (!mask || (mask[tok >> 5] >> (tok & 31) & 1)) g.bits |= 1u << e;
    }
  }
}

// The four count (or bias) words of a group: words [at, at + 4) of a shared array
// whose groups are aligned for shift 0 and lie `shift` words earlier otherwise; two
// aligned reads cover them.
DLLM_DEV void four_words(uint32_t (&r)[4], const uint32_t* a, int i, int shift) {
  const uint4 hi = *reinterpret_cast<const uint4*>(a + 4 * i + 4);
  if (shift == 0) {
    r[0] = hi.x, r[1] = hi.y, r[2] = hi.z, r[3] = hi.w;
    return;
  }
  const uint4 lo = *reinterpret_cast<const uint4*>(a + 4 * i);
  if (shift == 1)
    r[0] = lo.w, r[1] = hi.x, r[2] = hi.y, r[3] = hi.z;
  else if (shift == 2)
    r[0] = lo.z, r[1] = lo.w, r[2] = hi.x, r[3] = hi.y;
  else
    r[0] = lo.y, r[1] = lo.z, r[2] = lo.w, r[3] = hi.x;
}

// Grid (slices, row groups of a sequence, sequences). U: groups per thread and row,
// so a slice has 2048 U tokens.
template <int U>
__global__ void __launch_bounds__(kPickThreads, 2) pick_kernel(const PickArgs a, int rows) {
  constexpr int kSlice = kPickThreads * 4 * U;
  constexpr int kWords = kSlice + 4;  // a slice's tokens and the 4 before it (rows start up to 3 tokens early)
  extern __shared__ __align__(16) uint32_t dyn[];  // counts, then bias entries
  __shared__ unsigned long long warp_key[kMaxRowsPerCta][kPickWarps];
  const int tid = threadIdx.x, s = blockIdx.z;
  const int m = a.seqs ? a.seqs[s].m : 1;
  const int row0 = a.seqs ? a.seqs[s].row0 : s;
  const int r0 = blockIdx.y * rows, r1 = min(m, r0 + rows);
  if (r0 >= r1) return;
  const int c0 = blockIdx.x * kSlice;  // the slice: tokens [c0 - shift, c0 - shift + kSlice) of a row
  const int words = (a.vocab + 31) / 32;
  // a row's first group starts `shift` tokens before its slice, where its address is 16-byte aligned
  auto shift_of = [&](int row) { return (int)(((size_t)row * a.vocab) & 3); };
  auto mask_of = [&](int row) { return a.mask ? a.mask + (size_t)row * words : nullptr; };

  Group grp[U];
  {
    const int row = row0 + r0, sh = shift_of(row);
#pragma unroll
    for (int u = 0; u < U; ++u)
      load_group(grp[u], a.logits + (size_t)row * a.vocab, mask_of(row), c0 - sh + 4 * (tid + u * kPickThreads), a.vocab);
  }

  const bool counting = a.penalties != nullptr, biasing = a.bias_tok != nullptr;
  uint32_t* cnt = dyn;
  uint32_t* bia = counting ? dyn + kWords : dyn;
  RowRules r{1.f, 1.f, 1.f, nullptr};
  if (counting || biasing) {
    for (int i = tid; i < (counting + biasing) * kWords / 4; i += kPickThreads)
      reinterpret_cast<uint4*>(dyn)[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
  }
  if (counting) {
    r.rep = a.penalties[3 * s], r.freq = a.penalties[3 * s + 1], r.pres = a.penalties[3 * s + 2];
    if (a.hist) {
      const int h0 = clampi(a.hist_off[s], 0, a.hist_total), h1 = clampi(a.hist_off[s + 1], h0, a.hist_total);
      const int given = h0 + (a.prompt ? clampi(a.prompt[s], 0, h1 - h0) : 0);
      auto see = [&](int i, int tok) {  // ids outside the vocabulary fall outside every slice's rows
        const unsigned w = (unsigned)(tok - c0 + 4);
        if (w >= (unsigned)kWords) return;
        if (i < given)
          atomicOr(cnt + w, kGiven);
        else
          atomicAdd(cnt + w, 1u);
      };
      constexpr int B = 8;  // loads in flight
      for (int i = h0 + tid; i < h1; i += B * kPickThreads) {
        int tok[B];
#pragma unroll
        for (int e = 0; e < B; ++e) tok[e] = i + e * kPickThreads < h1 ? __ldg(a.hist + i + e * kPickThreads) : INT_MIN;
#pragma unroll
        for (int e = 0; e < B; ++e)
          if (tok[e] >= 0) see(i + e * kPickThreads, tok[e]);
      }
    }
  }
  if (biasing) {
    const int b0 = clampi(a.bias_off[s], 0, a.bias_total), b1 = clampi(a.bias_off[s + 1], b0, a.bias_total);
    r.bias_val = a.bias_val + b0;
    for (int i = b0 + tid; i < b1; i += kPickThreads) {
      const int tok = a.bias_tok[i];
      const unsigned w = (unsigned)(tok - c0 + 4);
      if (tok >= 0 && w < (unsigned)kWords) atomicMax(bia + w, (uint32_t)(i - b0 + 1));  // a token's last entry counts
    }
  }

  unsigned long long path = 0;  // nodes whose drafted tokens the counts hold
#pragma unroll 1
  for (int q = r0; q < r1; ++q) {
    const int row = row0 + q;
    if (counting && a.seqs) {
      const unsigned long long anc = a.anc[row];
      __syncthreads();  // the row before has been counted out
      if (tid < m && ((anc ^ path) >> tid & 1)) {
        const int tok = a.draft[row0 + tid];
        const unsigned w = (unsigned)(tok - c0 + 4);
        if (tok >= 0 && w < (unsigned)kWords) atomicAdd(cnt + w, (anc >> tid & 1) ? 1u : 0xffffffffu);
      }
      path = anc;
    }
    if (counting || biasing) __syncthreads();
    const int sh = shift_of(row), next = row + 1, nsh = shift_of(next);
    float* y = a.out ? a.out + (size_t)row * a.vocab : nullptr;
    Best best;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = tid + u * kPickThreads, t = c0 - sh + 4 * i;
      Group& g = grp[u];
      if (counting || biasing) {
        uint32_t k[4] = {0, 0, 0, 0}, b[4] = {0, 0, 0, 0};
        if (counting) four_words(k, cnt, i, sh);
        if (biasing) four_words(b, bia, i, sh);
        if (k[0] | k[1] | k[2] | k[3] | b[0] | b[1] | b[2] | b[3]) {
#pragma unroll
          for (int e = 0; e < 4; ++e) g.v[e] = apply(g.v[e], k[e], b[e], r);
        }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (g.bits >> e & 1)
          best.see(g.v[e], t + e);
        else
          g.v[e] = -INFINITY;
      }
      if (y) {
        if (t >= 0 && t + 3 < a.vocab) {
          __stcs(reinterpret_cast<float4*>(y + t), make_float4(g.v[0], g.v[1], g.v[2], g.v[3]));
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (t + e >= 0 && t + e < a.vocab) y[t + e] = g.v[e];
        }
      }
      if (q + 1 < r1)
        load_group(g, a.logits + (size_t)next * a.vocab, mask_of(next), c0 - nsh + 4 * i, a.vocab);
    }
    unsigned long long key = best.t < 0 ? 0ull : argmax_key(best.v, best.t);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const unsigned long long other = __shfl_xor_sync(0xffffffffu, key, o);
      if (other > key) key = other;
    }
    if ((tid & 31) == 0) warp_key[q - r0][tid >> 5] = key;
  }
  __syncthreads();
  if (tid < r1 - r0) {
    unsigned long long key = 0;
    for (int w = 0; w < kPickWarps; ++w) key = warp_key[tid][w] > key ? warp_key[tid][w] : key;
    const int row = row0 + r0 + tid;
    if (gridDim.x > 1) {
      if (key) atomicMax(a.best + row, key);
      __threadfence();
      if (atomicInc(a.arrived + row, gridDim.x - 1) != gridDim.x - 1) return;  // wraps to 0 with the last arrival
      __threadfence();
      key = atomicExch(a.best + row, 0ull);
    }
    a.tokens[row] = key ? argmax_key_index(key) : -1;
  }
}

// Processes rows [0, n) of `a` in one launch (n <= kPickMaxRows).
template <int U>
cudaError_t launch_pick(const PickArgs& a, int rows, int groups, int slices, cudaStream_t st) {
  const size_t smem = (size_t)(kPickThreads * 4 * U + 4) * 4 * ((a.penalties ? 1 : 0) + (a.bias_tok ? 1 : 0));
  pick_kernel<U><<<dim3(slices, groups, a.n_seqs), kPickThreads, smem, st>>>(a, rows);
  return cudaGetLastError();
}

}  // namespace

cudaError_t configure_pick_kernels() {
  return cudaFuncSetAttribute(pick_kernel<4>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                              2 * (kPickThreads * 16 + 4) * 4);
}

cudaError_t op_pick(const PickArgs& a, int sms, cudaStream_t st) {
  // Slices of 8192 tokens while they fill the SMs, else of 2048 (a single row over 75
  // CTAs instead of 19). A slice is reached by rows that start up to 3 tokens early,
  // hence vocab + 3. The nodes of a tree share a CTA as far as two CTAs per SM remain.
  const int wide = (a.vocab + 3 + 8191) / 8192, narrow = (a.vocab + 3 + 2047) / 2048;
  const long long ctas = (long long)a.n_seqs * a.max_m * wide;
  const int rows = (int)std::min<long long>(std::min(a.max_m, kMaxRowsPerCta), std::max<long long>(1, (ctas + 2 * sms - 1) / (2 * sms)));
  const int groups = (a.max_m + rows - 1) / rows;
  if (ctas >= sms) return launch_pick<4>(a, rows, groups, wide, st);
  return launch_pick<1>(a, rows, groups, narrow, st);
}

}  // namespace dllm
