// verify.cuh — host launchers of the kernels that verify drafted tokens: rotary
// positions per row (rope_at.cu), attention of a drafted tree over the paged
// cache (tree_attn.cu), token picks under penalties, biases and masks (pick.cu),
// and the cache rows of drafted tokens (tree_kv.cu).
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "common.cuh"

namespace dllm {

constexpr int kTreeMaxNodes = 64;  // nodes per sequence: one bit each of an ancestor mask
constexpr int kTreeMaxSeqs = 128;  // sequences per tree: their T0s travel as kernel arguments
constexpr int kErrTreeWait = 7;    // a tcgen05 attention kernel gave up waiting on an mbarrier

// One sequence of a drafted tree: its nodes are rows [row0, row0 + m) of the batch.
struct TreeSeq {
  int seq;  // sequence of the stage's cache
  int row0;
  int m;
  int pad;
};

// ---- rope_at.cu -----------------------------------------------------------------
struct RopeAtArgs {
  const float* q;  // [n][q_heads][hd], null with q_heads = 0
  const float* k;  // [n][k_heads][hd], null with k_heads = 0
  float* q_out;    // may be q itself
  float* k_out;
  const int32_t* pos;   // [n]
  const double* turns;  // [rotary / 2]: inverse frequency / 2 pi
  int n, q_heads, k_heads, hd, rotary, interleaved;
  float factor;
};
cudaError_t op_rope_at(const RopeAtArgs& a, int sms, cudaStream_t st);
struct NormRopeArgs {
  RopeAtArgs rope;
  const __nv_bfloat16* q_norm;  // [hd]
  const __nv_bfloat16* k_norm;
  float eps;
};
cudaError_t op_norm_rope(const NormRopeArgs& n, int sms, cudaStream_t st);

// ---- pick.cu ----------------------------------------------------------------------
struct PickArgs {
  const float* logits;  // [n][vocab]
  float* out;           // [n][vocab] or null
  int32_t* tokens;      // [n]
  int n, vocab;
  // token history of sequence s: tokens [hist_off[s], hist_off[s + 1]), then a node's path; the first
  // prompt[s] of them given
  const int32_t* hist;
  const int32_t* hist_off;
  const int32_t* prompt;
  int hist_total;
  const float* penalties;  // [n_seqs][3]: repetition, frequency, presence; null: none
  // additive biases of sequence s: entries [bias_off[s], bias_off[s + 1])
  const int32_t* bias_tok;
  const float* bias_val;
  const int32_t* bias_off;
  int bias_total;
  const uint32_t* mask;  // [n][ceil(vocab / 32)], bit set: allowed; null: everything
  // drafted tree: the rows of sequence s are its nodes; null: row i is sequence i
  const TreeSeq* seqs;
  const unsigned long long* anc;  // [n] ancestors (self included) within the sequence
  const int32_t* draft;           // [n] drafted tokens
  int n_seqs, max_m;
  // per row, zero before and after every call: the best key and the slices that have arrived
  unsigned long long* best;
  unsigned int* arrived;
};
constexpr int kPickMaxRows = kTreeMaxNodes * kTreeMaxSeqs;  // rows of one call (the capacity of best / arrived)
cudaError_t configure_pick_kernels();
cudaError_t op_pick(const PickArgs& a, int sms, cudaStream_t st);

// ---- tree_kv.cu ---------------------------------------------------------------------
struct TreeT0 {
  int t0[kTreeMaxSeqs];
};
// rows [n][kvh * hd] fp32 -> slots T0 + node of each sequence (rounded to the cache's type)
cudaError_t op_tree_append(const TreeSeq* seqs, int n_seqs, int max_m, const TreeT0& t0, const KvLayout& kv,
                           const float* k, const float* v, void* kc, void* vc, int kv_dtype, int kvh, int hd, int* err,
                           cudaStream_t st);
constexpr int kCommitSeqs = 32;  // sequences per launch
struct CommitArgs {
  int n_seqs;
  int seq[kCommitSeqs];
  int t0[kCommitSeqs];
  uint8_t first[kCommitSeqs];  // leading entries that stay where they are
  uint8_t len[kCommitSeqs];
  uint8_t path[kCommitSeqs][kTreeMaxNodes];
};
// slot t0 + path[j] -> slot t0 + j for j in [first, len), K and V of every layer
cudaError_t op_tree_commit(const CommitArgs& a, const KvLayout& kv, void* kpool, void* vpool, size_t layer_elems,
                           int layers, int kv_dtype, int kvh, int hd, cudaStream_t st);

// ---- tree_attn.cu -----------------------------------------------------------------------
struct TreeAttnArgs {
  const float* q;  // [n][nq][hd]
  float* out;      // [n][nq][hd]
  const void* kc;  // the layer's pools
  const void* vc;
  KvLayout kv;
  const unsigned long long* anc;
  int n_seqs, nq, kvh;
  float scale_log2;  // log2(e) / sqrt(hd)
  int* err;
  const void* tc_k;  // host: tensor maps (CUtensorMap) of the whole K and V pools as rows of hd
  const void* tc_v;
  int tc_row0;       // the layer's first row
  float* part_o;   // [slots][hd] partial outputs of sequences that are split
  float* part_ml;  // [slots][2]
};
// The call's sequences, on the host.
struct TreeAttnShape {
  const TreeSeq* seqs;
  const int* t0;  // [n_seqs]
  int n, max_m;
};
// Partial rows one call may write on `sms` SMs (the capacity of part_o / part_ml).
size_t tree_attn_part_rows(int sms);
cudaError_t configure_tree_attn();
cudaError_t op_tree_attention(const TreeAttnArgs& a, const TreeAttnShape& s, int kv_dtype, int hd, int sms,
                              int* launches, cudaStream_t st);

}  // namespace dllm
