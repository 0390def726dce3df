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
// First the history's tokens are counted, every slice's in its CTA's shared memory:
// the CTAs of a cluster share the reading and count into one another's memory (integer
// atomics, so their order does not matter). From then on nothing is written that
// another warp reads: a warp takes a row (or a part of one) through the slice's chunks,
// 4 tokens per lane, and applies the rules where a count word says so. A drafted token
// has the set of nodes that carry it, and its count for a node is the size of that set
// among the node's ancestors, less the nodes that a prompt longer than the history
// reaches. The slices' best (value, index) keys meet in one 64-bit atomicMax per row
// (the largest key wins in any order); the CTA that arrives last writes the tokens and
// clears the keys.
#include <cooperative_groups.h>

#include <algorithm>
#include <type_traits>

#include "verify.cuh"

namespace cg = cooperative_groups;

namespace dllm {
namespace {

constexpr int kPickThreads = 512;
constexpr int kPickWarps = kPickThreads / 32;
constexpr int kChunk = 128;       // tokens one warp covers at a time, 4 per lane
constexpr int kMaxChunks = 192;   // chunks per slice: two CTAs per SM have room for their count words, or for
                                  // half as many and the bias words
// Chunk c of a row has its tokens [128 c - shift, 128 c - shift + 128): a row whose
// address is `shift` elements past a 16-byte boundary starts that much early. So a
// chunk's words hold its 128 tokens behind the 4 before them, the last 3 of which are
// counted in two chunks.
constexpr int kLead = 4;
constexpr int kStride = kChunk + kLead;
constexpr int kCluster = 8;       // CTAs that share the reading of a history
constexpr int kSharedHistory = 8192;  // from this length on
constexpr int kBatch = 4;         // chunks whose loads are in flight together

constexpr uint32_t kGiven = 0x80000000u;    // the token occurs among the given (prompt) tokens
constexpr uint32_t kDrafted = 0x40000000u;  // the token is drafted somewhere in the tree
constexpr uint32_t kBiased = 0x20000000u;   // the token has a bias

struct RowRules {
  float rep, freq, pres;
  const float* bias_val;  // the sequence's bias entries
};

// The rules above for one token. cnt: its count word without kDrafted.
DLLM_DEV float apply(float x, uint32_t cnt, const uint32_t* bia, const RowRules& r) {
  const uint32_t c = cnt & ~(kGiven | kBiased);
  if (cnt & ~kBiased) x = x > 0.f ? __fdiv_rn(x, r.rep) : __fmul_rn(x, r.rep);
  if (c) x = __fsub_rn(__fsub_rn(x, __fmul_rn(r.freq, (float)c)), r.pres);
  if (cnt & kBiased) x = __fadd_rn(x, r.bias_val[*bia - 1]);
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
  unsigned long long given;                     // nodes whose tokens still belong to the prompt
  int32_t draft[kTreeMaxNodes];
  uint16_t drafted[2 * kTreeMaxNodes];          // words of drafted tokens
  int n_drafted;
  bool last;
};

// The four count words of a lane's group, which starts `sh` words before an aligned place:
// two aligned reads cover them.
template <bool ALIGNED>
DLLM_DEV void four_words(uint32_t (&r)[4], const uint32_t* p, int sh) {
  const uint4 hi = *reinterpret_cast<const uint4*>(p);
  r[0] = hi.x, r[1] = hi.y, r[2] = hi.z, r[3] = hi.w;
  if (ALIGNED || sh == 0) return;
  const uint4 lo = *reinterpret_cast<const uint4*>(p - 4);
  if (sh == 1)
    r[3] = hi.z, r[2] = hi.y, r[1] = hi.x, r[0] = lo.w;
  else if (sh == 2)
    r[3] = hi.y, r[2] = hi.x, r[1] = lo.w, r[0] = lo.z;
  else
    r[3] = hi.x, r[2] = lo.w, r[1] = lo.z, r[0] = lo.y;
}

// Grid (K slices, sequences), K = 1 << log2k: slice s has the chunks c with c % K = s,
// n_chunks of them at most. Clusters of neighbouring slices. ALIGNED: the vocabulary is a
// multiple of 4, so every row starts at a 16-byte boundary.
// PROMPTED: a tree with prompt lengths.
template <bool ALIGNED, bool PROMPTED>
__global__ void __launch_bounds__(kPickThreads, 2) pick_kernel(const PickArgs a, int log2k, int n_chunks) {
  extern __shared__ __align__(16) uint32_t dyn[];  // counts, and bias entries if there are any, of the slice's words
  __shared__ PickShared sm;
  cg::cluster_group cluster = cg::this_cluster();
  const unsigned csize = cluster.num_blocks(), crank = cluster.block_rank();
  const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
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
  // the loads of kBatch chunks of a row, from chunk lc0 on
  Group grp[kBatch];
  auto load_chunks = [&](int q, int lc0) {
    const int row = row0 + q, sh = ALIGNED ? 0 : (int)(((size_t)row * a.vocab) & 3);
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const int lc = lc0 + u * parts;
      if (lc < n_chunks)
        load_group<ALIGNED>(grp[u], a.logits + (size_t)row * a.vocab, a.mask ? a.mask + (size_t)row * mask_words : nullptr,
                            token_of(lc) - sh, a.vocab);
    }
  };
  if (first_row < min(n_rows, m)) load_chunks(first_row, part);  // on their way while the history is counted

  const bool counting = a.penalties != nullptr, biasing = a.bias_tok != nullptr, ruled = counting || biasing;
  const bool pathed = counting && a.seqs;
  uint32_t* cnt = dyn;
  uint32_t* bia = dyn + n_words;
  RowRules r{1.f, 1.f, 1.f, nullptr};
  // what the counting needs first is loaded before the shared memory is cleared
  constexpr int B = 8;  // history loads in flight per thread
  const int h_step = (int)csize * kPickThreads;
  int h0 = 0, h1 = 0, given = 0, levels = 0, b0 = 0, b1 = 0, tok[B];
  if (counting) {
    r.rep = a.penalties[3 * s], r.freq = a.penalties[3 * s + 1], r.pres = a.penalties[3 * s + 2];
    if (a.hist) {
      const int o0 = a.hist_off[s], o1 = a.hist_off[s + 1], pl = a.prompt ? a.prompt[s] : 0;
      h0 = clampi(o0, 0, a.hist_total), h1 = clampi(o1, h0, a.hist_total), given = h0 + clampi(pl, 0, h1 - h0);
      if (PROMPTED && pl > h1 - h0) levels = pl - (h1 - h0);  // of the tree, which the prompt reaches into
    }
  }
  if (biasing) {
    const int o0 = a.bias_off[s], o1 = a.bias_off[s + 1];
    b0 = clampi(o0, 0, a.bias_total), b1 = clampi(o1, b0, a.bias_total);
    r.bias_val = a.bias_val + b0;
  }
  auto load_history = [&](int i) {
#pragma unroll
    for (int e = 0; e < B; ++e) tok[e] = i + e * h_step < h1 ? __ldg(a.hist + i + e * h_step) : -1;
  };
  int h_at = h0 + (int)crank * kPickThreads + tid;
  load_history(h_at);
  const int b_tok = b0 + tid < b1 ? a.bias_tok[b0 + tid] : -1;
  if (tid < kTreeMaxNodes) sm.key[tid] = 0ull;
  if (tid == 0) {
    sm.n_drafted = 0;
    if (PROMPTED) sm.given = 0ull;
  }
  if (ruled) {
    for (int i = tid; i < (biasing ? 2 : 1) * n_words / 4; i += kPickThreads) reinterpret_cast<uint4*>(dyn)[i] = make_uint4(0, 0, 0, 0);
    if (pathed && tid < m) sm.draft[tid] = a.draft[row0 + tid];
  }
  if (csize > 1)
    cluster.sync();
  else
    __syncthreads();
  // calls f(slice, word) for the words of a token within the `span` slices from `from` (a
  // multiple of the power of two `span`): its own, and the one of the next chunk if rows
  // can start early enough to have it there
  auto words_of = [&](int tok, unsigned from, unsigned span, auto f) {
    const unsigned c = (unsigned)tok / kChunk, in = tok & (kChunk - 1), near = kmask & ~(span - 1);
    if (((c ^ from) & near) == 0 && (unsigned)tok < (unsigned)a.vocab) f(c & kmask, (int)((c >> log2k) * kStride + kLead + in));
    if (!ALIGNED && in >= kChunk - 3 && (((c + 1) ^ from) & near) == 0 && (unsigned)tok < (unsigned)a.vocab &&
        (c + 1) >> log2k < (unsigned)n_chunks)
      f((c + 1) & kmask, (int)(((c + 1) >> log2k) * kStride + kLead + in - kChunk));
  };
  if (counting) {
    while (h_at < h1) {
#pragma unroll
      for (int e = 0; e < B; ++e) {
        if (tok[e] < 0) continue;
        words_of(tok[e], slice & ~(csize - 1), csize, [&](unsigned sl, int w) {
          uint32_t* to = csize > 1 ? cluster.map_shared_rank(cnt, sl & (csize - 1)) : cnt;
          if (h_at + e * h_step < given)
            atomicOr(to + w, kGiven);
          else
            atomicAdd(to + w, 1u);
        });
      }
      h_at += B * h_step;
      load_history(h_at);
    }
    if (pathed && tid < m) {
      words_of(sm.draft[tid], slice, 1, [&](unsigned, int w) {
        if (!(atomicOr(cnt + w, kDrafted) & kDrafted)) sm.drafted[atomicAdd(&sm.n_drafted, 1)] = (uint16_t)w;
      });
      if (PROMPTED && levels && __popcll(a.anc[row0 + tid]) <= levels) atomicOr(&sm.given, 1ull << tid);
    }
  }
  for (int i = b0 + tid; i < b1; i += kPickThreads)
    words_of(i == b0 + tid ? b_tok : a.bias_tok[i], slice, 1, [&](unsigned, int w) {
      atomicOr(cnt + w, kBiased);
      atomicMax(bia + w, (uint32_t)(i - b0 + 1));  // of a token listed twice the last entry counts
    });
  if (ruled) {
    if (csize > 1)
      cluster.sync();
    else
      __syncthreads();
    if (tid < sm.n_drafted) {
      const int w = sm.drafted[tid], lc = w / kStride;
      const int tok = ((lc << log2k) + slice) * kChunk + (w - lc * kStride) - kLead;
      unsigned long long nodes = 0;
      for (int j = 0; j < m; ++j) nodes |= (unsigned long long)(sm.draft[j] == tok) << j;
      sm.nodes[tid] = nodes;
    }
    if (pathed) __syncthreads();
  }

  // A prompt that reaches into the tree is rare: its rule has a copy of the loop of its own
  // (in the one loop it cost 64 nodes of 152064 tokens 5 %), in trees with prompt lengths only
  // (16 rows of 50257 took 12.3 us with the copy, 12.0 without).
  auto rows = [&](auto with_given) {
    constexpr bool GIVEN = decltype(with_given)::value;
#pragma unroll 1
    for (int q = first_row; q < m && first_row < n_rows; q += n_rows) {
      const int row = row0 + q, sh = ALIGNED ? 0 : (int)(((size_t)row * a.vocab) & 3);
      float* y = a.out ? a.out + (size_t)row * a.vocab : nullptr;
      const uint32_t* mask = a.mask ? a.mask + (size_t)row * mask_words : nullptr;
      const unsigned long long anc = pathed ? a.anc[row] : 0ull;
      float bv = -INFINITY;  // the greatest allowed logit of this lane, and its first token
      int bt = -1;
#pragma unroll 1
      for (int lc0 = part; lc0 < n_chunks; lc0 += kBatch * parts) {
        if (lc0 != part || q != first_row) load_chunks(q, lc0);
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
          const int lc = lc0 + u * parts, t = token_of(lc) - sh;
          if (lc >= n_chunks) break;
          Group& g = grp[u];
          if (ruled) {
            const int w = lc * kStride + kLead - sh + 4 * lane;
            uint32_t c[4];
            four_words<ALIGNED>(c, cnt + w + sh, sh);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              if (!(g.bits >> e & 1)) c[e] = 0;
              if (c[e] & kDrafted) {
                int d = 0;
                while (sm.drafted[d] != w + e) ++d;
                const unsigned long long on = anc & sm.nodes[d];
                c[e] = (c[e] & ~kDrafted) + (uint32_t)__popcll(GIVEN ? on & ~sm.given : on);
                if (GIVEN && (on & sm.given)) c[e] |= kGiven;
              }
              if (c[e]) g.v[e] = apply(g.v[e], c[e], bia + w + e, r);
            }
          }
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (!(g.bits >> e & 1)) g.v[e] = -INFINITY;
          if (y) store_group<ALIGNED>(y, g, t, a.vocab);
          const float most = fmaxf(fmaxf(g.v[0], g.v[1]), fmaxf(g.v[2], g.v[3]));  // passes over NaN
          if (most > bv) {
            bv = most;
            bt = t + (g.v[0] == most ? 0 : g.v[1] == most ? 1 : g.v[2] == most ? 2 : 3);
          }
        }
      }
      // a lane without a logit above -inf (or only NaN): its first allowed token counts as -inf
      if (bt < 0) {
        for (int lc = part; lc < n_chunks && bt < 0; lc += parts) {
          const int t = token_of(lc) - sh;
          for (int e = 3; e >= 0; --e)
            if (t + e >= 0 && t + e < a.vocab && (!mask || (mask[(t + e) >> 5] >> ((t + e) & 31) & 1))) bt = t + e;
        }
      }
      // the warp's best: the greatest value, then the lowest token (-0 + 0 = +0: zeros tie)
      const uint32_t bits = __float_as_uint(__fadd_rn(bv, 0.f)), ord = bt < 0 ? 0u : (bits & 0x80000000u) ? ~bits : bits | 0x80000000u;
      const uint32_t top = __reduce_max_sync(0xffffffffu, ord);
      const uint32_t tok = __reduce_min_sync(0xffffffffu, ord == top && bt >= 0 ? (uint32_t)bt : 0xffffffffu);
      const unsigned long long key = top ? ((unsigned long long)top << 32) | ~tok : 0ull;
      if (lane == 0 && key) atomicMax(&sm.key[q], key);
    }
  };
  if (PROMPTED && pathed && sm.given)
    rows(std::bool_constant<PROMPTED>());
  else
    rows(std::false_type());
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

constexpr size_t pick_smem(int n_chunks) { return (size_t)n_chunks * kStride * 4; }  // one set of words

}  // namespace

cudaError_t configure_pick_kernels() {
  const int smem = (int)pick_smem(kMaxChunks);
  for (auto* kernel : {pick_kernel<true, true>, pick_kernel<true, false>, pick_kernel<false, true>, pick_kernel<false, false>}) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

cudaError_t op_pick(const PickArgs& a, int sms, cudaStream_t st) {
  // The fewest slices whose count words fit a CTA (one without rules, which has none), then
  // twice as many as long as all CTAs still run at once, two per SM, and a slice keeps at
  // least 4 chunks and one for every warp. A row that starts 3 tokens early reaches vocab + 3.
  const long long chunks = ((long long)a.vocab + 3 + kChunk - 1) / kChunk;
  int log2k = 0;
  const int sets = (a.penalties || a.bias_tok ? 1 : 0) + (a.bias_tok ? 1 : 0);
  while ((chunks + (1ll << log2k) - 1) * sets >> log2k > kMaxChunks) ++log2k;
  while ((2ll << log2k) * a.n_seqs <= 2ll * sms && chunks >> (log2k + 1) >= 4 &&
         (chunks >> (log2k + 1)) * a.max_m >= kPickWarps)
    ++log2k;
  const int n_chunks = (int)((chunks + (1ll << log2k) - 1) >> log2k);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(1u << log2k, a.n_seqs);
  cfg.blockDim = dim3(kPickThreads);
  cfg.dynamicSmemBytes = sets * pick_smem(n_chunks);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  // A cluster costs two cluster barriers: worth it from about 8000 tokens per history
  // (launches back to back: one row over 1500 tokens takes 2.6 us more with them; 64 nodes
  // over 32000 take 39 us, 45 without). The histories' lengths are on the device: the rule
  // takes the buffer's.
  attr[0].val.clusterDim.x = a.hist_total / a.n_seqs >= kSharedHistory ? std::min(kCluster, 1 << log2k) : 1;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const bool prompted = a.seqs && a.prompt;
  return cudaLaunchKernelEx(&cfg,
                            a.vocab % 4 == 0 ? (prompted ? pick_kernel<true, true> : pick_kernel<true, false>)
                                             : (prompted ? pick_kernel<false, true> : pick_kernel<false, false>),
                            a, log2k, n_chunks);
}

}  // namespace dllm
