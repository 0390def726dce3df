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
// sequence, that is one row, or all nodes of a tree, which share their history. The
// slice is every K-th chunk of 128 tokens, not a contiguous range: text uses low token
// ids far more often, and the CTA with the first tokens would hold half the history.
// First the CTA counts the history's tokens that fall into its slice in shared memory
// (integer atomics, so their order does not matter) and flags the tokens that any rule
// touches, one bit each. From then on nothing is written that another warp reads: a warp
// takes a row (or a part of one) through the slice's chunks, 4 tokens per lane. The
// flagged tokens of a group are worked off one per lane and round, which keeps the
// divisions to about two rounds where one token in ten is flagged instead of four. A
// drafted token has the set of nodes that carry it, and its count for a node is the
// size of that set among the node's ancestors. The slices' best (value, index) keys meet
// in one 64-bit atomicMax per row (the largest key wins in any order); the CTA that
// arrives last writes the tokens and clears the keys.
#include <algorithm>

#include "verify.cuh"

namespace dllm {
namespace {

constexpr int kPickThreads = 512;
constexpr int kPickWarps = kPickThreads / 32;
constexpr int kChunk = 128;       // tokens one warp covers at a time, 4 per lane
constexpr int kMaxChunks = 64;    // chunks per slice
// Chunk c of a row has its tokens [128 c - shift, 128 c - shift + 128): a row whose
// address is `shift` elements past a 16-byte boundary starts that much early. So a
// chunk's words hold its 128 tokens behind a lead of 32, whose last 3 are the tokens
// before it (they are counted in two chunks); with a lead of 32 the flags of a lane's
// group lie in one word when shift is 0.
constexpr int kLead = 32;
constexpr int kStride = kChunk + kLead;
constexpr int kMaxFlags = kMaxChunks * kStride / 32;
constexpr int kBatch = 4;         // chunks whose loads are in flight together

constexpr uint32_t kGiven = 0x80000000u;    // the token occurs among the given (prompt) tokens
constexpr uint32_t kDrafted = 0x40000000u;  // the token is drafted somewhere in the tree

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

// One lane's 16-byte group of a row: tokens [t, t + 4). At a row's ends some of them may
// lie outside the vocabulary (rows whose length is no multiple of 4 start inside a
// group). bits: which of the four are allowed tokens.
struct Group {
  float v[4];
  uint32_t bits;
};

// ALIGNED rows have groups that lie within the vocabulary or behind it as a whole, and
// their mask bits lie in one word.
template <bool ALIGNED>
DLLM_DEV void load_group(Group& g, const float* x, const uint32_t* mask, int t, int vocab) {
  g.bits = 0xfu;
  if (ALIGNED ? t < vocab : t >= 0 && t + 3 < vocab) {
    const float4 f = __ldcs(reinterpret_cast<const float4*>(x + t));
    g.v[0] = f.x, g.v[1] = f.y, g.v[2] = f.z, g.v[3] = f.w;
    if (mask) {
      const int sh = t & 31;
      g.bits = __ldg(mask + (t >> 5)) >> sh;
      if (!ALIGNED && sh > 28) g.bits |= __ldg(mask + (t >> 5) + 1) << (32 - sh);
      g.bits &= 0xfu;
    }
    return;
  }
  if constexpr (ALIGNED) {
    g.bits = 0;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int tok = t + e;
      const bool in = tok >= 0 && tok < vocab;
      g.v[e] = in ? x[tok] : 0.f;
      if (!in || (mask && !(mask[tok >> 5] >> (tok & 31) & 1))) g.bits &= ~(1u << e);
    }
  }
}

template <bool ALIGNED>
DLLM_DEV void store_group(float* y, const Group& g, int t, int vocab) {
  if (ALIGNED ? t < vocab : t >= 0 && t + 3 < vocab) {
    __stcs(reinterpret_cast<float4*>(y + t), make_float4(g.v[0], g.v[1], g.v[2], g.v[3]));
  } else if (!ALIGNED) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (t + e >= 0 && t + e < vocab) y[t + e] = g.v[e];
  }
}

struct PickShared {
  unsigned long long key[kTreeMaxNodes];
  unsigned long long nodes[2 * kTreeMaxNodes];  // per entry of drafted: the nodes with that token
  uint32_t flag[kMaxFlags + 1];                 // bit w: a rule touches the token of word w
  int32_t draft[kTreeMaxNodes];
  uint16_t drafted[2 * kTreeMaxNodes];          // words of drafted tokens
  int n_drafted;
  bool last;
};

// Grid (K slices, sequences), K = 1 << log2k: slice s has the chunks c with c % K = s,
// n_chunks of them at most. ALIGNED: the vocabulary is a multiple of 4, so every row is.
template <bool ALIGNED>
__global__ void __launch_bounds__(kPickThreads, 2) pick_kernel(const PickArgs a, int log2k, int n_chunks) {
  extern __shared__ __align__(16) uint32_t dyn[];  // counts, bias entries of the slice's words
  __shared__ PickShared sm;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int slice = blockIdx.x, s = blockIdx.y;
  const int m = a.seqs ? a.seqs[s].m : 1;
  const int row0 = a.seqs ? a.seqs[s].row0 : s;
  if (m == 0) return;
  const int n_words = n_chunks * kStride;
  const int mask_words = (a.vocab + 31) / 32;
  const unsigned kmask = (1u << log2k) - 1;
  auto token_of = [&](int lc) { return ((lc << log2k) + slice) * kChunk + 4 * lane; };

  // warps: `parts` of them share a row, n_rows rows are under way at once
  const int parts = m < kPickWarps ? kPickWarps / m : 1, n_rows = kPickWarps / parts;
  const int part = warp % parts, first_row = warp / parts;
  // asks L2 for this warp's part of a row while something else is done
  auto fetch = [&](int q) {
    if (q >= m || first_row >= n_rows) return;
    const float* x = a.logits + (size_t)(row0 + q) * a.vocab;
    for (int lc = part; lc < n_chunks; lc += parts) {
      const int t = token_of(lc);
      if (t < a.vocab) asm volatile("prefetch.global.L2 [%0];" ::"l"(x + t));
    }
  };
  fetch(first_row);

  const bool counting = a.penalties != nullptr, biasing = a.bias_tok != nullptr, ruled = counting || biasing;
  const bool pathed = counting && a.seqs;
  uint32_t* cnt = dyn;
  uint32_t* bia = dyn + n_words;
  RowRules r{1.f, 1.f, 1.f, nullptr};
  if (tid < kTreeMaxNodes) sm.key[tid] = 0ull;
  if (tid == 0) sm.n_drafted = 0;
  if (ruled) {
    for (int i = tid; i < 2 * n_words / 4; i += kPickThreads) reinterpret_cast<uint4*>(dyn)[i] = make_uint4(0, 0, 0, 0);
    if (pathed && tid < m) sm.draft[tid] = a.draft[row0 + tid];
  }
  __syncthreads();
  // calls f(word) for the words of a token within the slice: its own, and the one of the
  // next chunk if rows can start early enough to have it there
  auto words_of = [&](int tok, auto f) {
    const unsigned c = (unsigned)tok / kChunk, in = tok & (kChunk - 1);
    if (((c ^ slice) & kmask) == 0 && (unsigned)tok < (unsigned)a.vocab) f((c >> log2k) * kStride + kLead + in);
    if (!ALIGNED && in >= kChunk - 3 && (((c + 1) ^ slice) & kmask) == 0 && (unsigned)tok < (unsigned)a.vocab &&
        (c + 1) >> log2k < (unsigned)n_chunks)
      f(((c + 1) >> log2k) * kStride + kLead + in - kChunk);
  };
  if (counting) {
    r.rep = a.penalties[3 * s], r.freq = a.penalties[3 * s + 1], r.pres = a.penalties[3 * s + 2];
    if (a.hist) {
      const int h0 = clampi(a.hist_off[s], 0, a.hist_total), h1 = clampi(a.hist_off[s + 1], h0, a.hist_total);
      const int given = h0 + (a.prompt ? clampi(a.prompt[s], 0, h1 - h0) : 0);
      auto see = [&](int i, int tok) {
        words_of(tok, [&](int w) {
          if (i < given)
            atomicOr(cnt + w, kGiven);
          else
            atomicAdd(cnt + w, 1u);
        });
      };
      // Every CTA reads the whole history: each starts at a place of its own, so that they
      // do not all ask the same L2 slice for the same line (18k cycles for 32000 tokens
      // in step, 256 CTAs).
      constexpr int B = 16;  // loads in flight
      const int span = B * kPickThreads, turns = (h1 - h0 + span - 1) / span;
      for (int n = 0, turn = turns ? slice % turns : 0; n < turns; ++n, turn = turn + 1 < turns ? turn + 1 : 0) {
        const int i = h0 + turn * span + tid;
        int tok[B];
#pragma unroll
        for (int e = 0; e < B; ++e) tok[e] = i + e * kPickThreads < h1 ? __ldg(a.hist + i + e * kPickThreads) : -1;
#pragma unroll
        for (int e = 0; e < B; ++e) see(i + e * kPickThreads, tok[e]);
      }
    }
    if (pathed && tid < m)
      words_of(sm.draft[tid], [&](int w) {
        if (!(atomicOr(cnt + w, kDrafted) & kDrafted)) sm.drafted[atomicAdd(&sm.n_drafted, 1)] = (uint16_t)w;
      });
  }
  if (biasing) {
    const int b0 = clampi(a.bias_off[s], 0, a.bias_total), b1 = clampi(a.bias_off[s + 1], b0, a.bias_total);
    r.bias_val = a.bias_val + b0;
    for (int i = b0 + tid; i < b1; i += kPickThreads)
      words_of(a.bias_tok[i], [&](int w) { atomicMax(bia + w, (uint32_t)(i - b0 + 1)); });  // the last entry counts
  }
  if (ruled) {
    __syncthreads();
    for (int w = tid; w < n_words; w += kPickThreads) {  // whole warps: n_words is a multiple of 32
      const uint32_t any = __ballot_sync(0xffffffffu, cnt[w] | bia[w]);
      if (lane == 0) sm.flag[w >> 5] = any;
    }
    if (tid == 0) sm.flag[n_words / 32] = 0u;
    if (tid < sm.n_drafted) {
      const int w = sm.drafted[tid], lc = w / kStride;
      const int tok = ((lc << log2k) + slice) * kChunk + (w - lc * kStride) - kLead;
      unsigned long long nodes = 0;
      for (int j = 0; j < m; ++j) nodes |= (unsigned long long)(sm.draft[j] == tok) << j;
      sm.nodes[tid] = nodes;
    }
    __syncthreads();
  }

#pragma unroll 1
  for (int q = first_row; q < m && first_row < n_rows; q += n_rows) {
    const int row = row0 + q, sh = ALIGNED ? 0 : (int)(((size_t)row * a.vocab) & 3);
    const float* x = a.logits + (size_t)row * a.vocab;
    float* y = a.out ? a.out + (size_t)row * a.vocab : nullptr;
    const uint32_t* mask = a.mask ? a.mask + (size_t)row * mask_words : nullptr;
    const unsigned long long anc = pathed ? a.anc[row] : 0ull;
    float bv = -INFINITY;  // best of this lane: the first allowed token, then whatever is greater
    int bt = -1;
#pragma unroll 1
    for (int lc0 = part; lc0 < n_chunks; lc0 += kBatch * parts) {
      Group grp[kBatch];
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const int lc = lc0 + u * parts;
        if (lc < n_chunks) load_group<ALIGNED>(grp[u], x, mask, token_of(lc) - sh, a.vocab);
      }
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const int lc = lc0 + u * parts, t = token_of(lc) - sh;
        if (lc >= n_chunks) break;
        Group& g = grp[u];
        if (ruled) {
          const int w = lc * kStride + kLead - sh + 4 * lane;
          uint32_t touched = sm.flag[w >> 5] >> (w & 31);
          if (!ALIGNED) touched = __funnelshift_r(sm.flag[w >> 5], sm.flag[(w >> 5) + 1], w & 31);
          touched &= g.bits;
          while (touched) {  // one token per lane and round
            const int e = __ffs(touched) - 1;
            touched &= touched - 1;
            uint32_t c = cnt[w + e];
            if (c & kDrafted) {
              int d = 0;
              while (sm.drafted[d] != w + e) ++d;
              c = (c & ~kDrafted) + (uint32_t)__popcll(anc & sm.nodes[d]);
            }
            const float old = e == 0 ? g.v[0] : e == 1 ? g.v[1] : e == 2 ? g.v[2] : g.v[3];
            const float z = apply(old, c, bia[w + e], r);
            g.v[0] = e == 0 ? z : g.v[0];
            g.v[1] = e == 1 ? z : g.v[1];
            g.v[2] = e == 2 ? z : g.v[2];
            g.v[3] = e == 3 ? z : g.v[3];
          }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (!(g.bits >> e & 1)) g.v[e] = -INFINITY;
        if (y) store_group<ALIGNED>(y, g, t, a.vocab);
        const float most = fmaxf(fmaxf(g.v[0], g.v[1]), fmaxf(g.v[2], g.v[3]));  // NaN counts as -inf
        if (most > bv || (bt < 0 && g.bits)) {
#pragma unroll
          for (int e = 3; e >= 0; --e)
            if ((g.bits >> e & 1) && (g.v[e] == most || !(most > -INFINITY))) bt = t + e;
          bv = most == most ? most : -INFINITY;
        }
      }
    }
    unsigned long long key = bt < 0 ? 0ull : argmax_key(bv, bt);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const unsigned long long other = __shfl_xor_sync(0xffffffffu, key, o);
      if (other > key) key = other;
    }
    if (lane == 0 && key) atomicMax(&sm.key[q], key);
  }
  __syncthreads();
  if (gridDim.x > 1) {
    if (tid < m && sm.key[tid]) atomicMax(a.best + row0 + tid, sm.key[tid]);
    __threadfence();
    __syncthreads();
    if (tid == 0) sm.last = atomicInc(a.arrived + s, gridDim.x - 1) == gridDim.x - 1;  // wraps to 0 with the last
    __syncthreads();
    if (!sm.last) return;
    __threadfence();
    if (tid < m) sm.key[tid] = atomicExch(a.best + row0 + tid, 0ull);
  }
  if (tid < m) a.tokens[row0 + tid] = sm.key[tid] ? argmax_key_index(sm.key[tid]) : -1;
}

// counts and bias entries of a slice's words
constexpr size_t pick_smem(int n_chunks) { return (size_t)n_chunks * kStride * 8; }

}  // namespace

cudaError_t configure_pick_kernels() {
  const int smem = (int)pick_smem(kMaxChunks);
  cudaError_t e = cudaFuncSetAttribute(pick_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e == cudaSuccess) e = cudaFuncSetAttribute(pick_kernel<false>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  return e;
}

cudaError_t op_pick(const PickArgs& a, int sms, cudaStream_t st) {
  // The fewest slices that fit a CTA (64 chunks), then twice as many as long as all CTAs
  // still run at once, two per SM, and a slice keeps at least 4 chunks. A row that starts 3
  // tokens early reaches vocab + 3.
  const long long chunks = ((long long)a.vocab + 3 + kChunk - 1) / kChunk;
  int log2k = 0;
  while ((chunks + (1ll << log2k) - 1) >> log2k > kMaxChunks) ++log2k;
  while ((2ll << log2k) * a.n_seqs <= 2ll * sms && chunks >> (log2k + 1) >= 4) ++log2k;
  const int n_chunks = (int)((chunks + (1ll << log2k) - 1) >> log2k);
  const size_t smem = a.penalties || a.bias_tok ? pick_smem(n_chunks) : 0;
  const dim3 grid(1u << log2k, a.n_seqs);
  if (a.vocab % 4 == 0)
    pick_kernel<true><<<grid, kPickThreads, smem, st>>>(a, log2k, n_chunks);
  else
    pick_kernel<false><<<grid, kPickThreads, smem, st>>>(a, log2k, n_chunks);
  return cudaGetLastError();
}

}  // namespace dllm
