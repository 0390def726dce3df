/*
 * dllm.h — C ABI of libdllm.so, the B200 (sm_100a) decode path for Qwen2.5-style
 * decoders.
 *
 * The entry points mirror the JavaScript surface that the reference's decode loop
 * sits behind, so a host binding (N-API, ctypes, cgo ...) can swap the WebGPU path
 * for this library one call at a time:
 *   - kernels.js  `initKernels(device)` -> ctx with buffer helpers and op launchers
 *   - pipeline.js `Stage` (layer range + KV cache) and `LeaderPipeline`
 *   - weights.js  bf16 weight layout (raw bits, one element per u32 on the JS side)
 * Every function cites the reference interface it replaces as file:line.
 *
 * Conventions
 *   - Every call returns a status (DLLM_OK == 0); on error `dllm_last_error(ctx)`
 *     holds a one-line message. The JS shim turns a non-zero status into
 *     `throw new Error(msg)`, as the reference throws (kernels.js:182,189,196,244).
 *   - One host thread per ctx; calls are not re-entrant. Work is enqueued on the
 *     ctx's CUDA stream; only calls that hand data back to the host synchronise,
 *     and those waits are bounded (DLLM_ETIMEOUT), mirroring readF32's 15 s limit
 *     (kernels.js:201-207).
 *   - Buffers are reference counted. The caller owns every dllm_buf it receives
 *     and releases it with dllm_buf_free; a stage that is given a weight buffer
 *     keeps its own reference (JS keeps the GPUBuffer alive the same way).
 *   - Activations are fp32 and weights bf16, as in the reference. The KV cache is
 *     fp32 (the reference's precision) or bf16 (half the bytes), chosen per ctx.
 */
#ifndef DLLM_H
#define DLLM_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* ---- status codes ---------------------------------------------------------- */
enum {
  DLLM_OK = 0,
  DLLM_EINVAL = 1,    /* bad argument: the reference throws "invalid size" (kernels.js:182,189,196,244) */
  DLLM_ENOMEM = 2,    /* device allocation failed */
  DLLM_ERANGE = 3,    /* KV cache overflow: T0 + n > max_pos (pipeline.js:38-43 sizes the cache) */
  DLLM_ETIMEOUT = 4,  /* bounded wait expired (readF32 15 s, kernels.js:201-207) */
  DLLM_ECUDA = 5,     /* CUDA runtime error */
  DLLM_ENOTFOUND = 6, /* missing weight tensor name (Stage.W lookup, pipeline.js:55-73) */
  DLLM_EDEVICE = 7    /* a kernel reported an error status (device-side bounds check) */
};

enum { DLLM_KV_F32 = 0, DLLM_KV_BF16 = 1 };

/* Model and cache configuration. Replaces the hard-coded CFG object of
 * constants.js:10-23 and the dims baked into the shaders (kernels.js:173). */
typedef struct dllm_config {
  int32_t vocab_size;          /* CFG.vocabSize */
  int32_t hidden_size;         /* CFG.hiddenSize (D) */
  int32_t num_layers;          /* CFG.numLayers */
  int32_t num_q_heads;         /* CFG.numQHeads (NQ) */
  int32_t num_kv_heads;        /* CFG.numKVHeads (KVH) */
  int32_t head_dim;            /* CFG.headDim (HD): 64 or 128 */
  int32_t intermediate_size;   /* CFG.intermediateSize */
  float rope_theta;            /* CFG.ropeTheta */
  float rms_norm_eps;          /* CFG.rmsNormEps */
  int32_t tie_word_embeddings; /* CFG.tieWordEmbeddings: LM head = embed_tokens */
  int32_t eos_token_id;        /* CFG.eosTokenId */
  int32_t max_pos;             /* CFG.maxPos: KV slots per sequence */
  int32_t kv_dtype;            /* DLLM_KV_F32 (reference precision) or DLLM_KV_BF16 */
  int32_t kv_page_size;        /* KV slots per page, power of two (paged cache) */
  int32_t max_seqs;            /* sequences one stage holds KV for (micro-batching) */
} dllm_config;

typedef struct dllm_ctx dllm_ctx;
typedef struct dllm_buf dllm_buf;
typedef struct dllm_stage dllm_stage;
typedef struct dllm_leader dllm_leader;

/* ---- library / context ----------------------------------------------------- */
const char* dllm_version(void);
const char* dllm_status_string(int status);
/* Text of a code that a kernel left in an error flag (dllm_attention_noalloc_status). */
const char* dllm_device_error_string(int code);
/* Fills the Qwen2.5-1.5B defaults of constants.js:10-23 (max_pos 4096, fp32 KV). */
void dllm_config_default(dllm_config* cfg);

/* initKernels(device) -> ctx (kernels.js:5,179). `device` is a CUDA ordinal. */
int dllm_init_kernels(int device, const dllm_config* cfg, dllm_ctx** out);
void dllm_ctx_destroy(dllm_ctx* ctx);
const char* dllm_last_error(const dllm_ctx* ctx);
int dllm_ctx_get_config(const dllm_ctx* ctx, dllm_config* out);
/* Enqueue on a caller-owned cudaStream_t (NULL restores the ctx's own stream). */
int dllm_ctx_set_stream(dllm_ctx* ctx, void* cuda_stream);
/* Bounded wait for all work on the ctx stream (timeout_ms <= 0: 15000 ms). */
int dllm_ctx_synchronize(dllm_ctx* ctx, int timeout_ms);
/* Number of kernels this ctx has launched (host counter, for launch accounting). */
uint64_t dllm_ctx_launch_count(const dllm_ctx* ctx);
/* Passes of at least `min_rows` rows (MATMUL with n > 1, kernels.js:26-44; prefill
 * chunks and wide micro-batches of Stage.forward, pipeline.js:48-78) run their
 * projections as tcgen05 tensor-core GEMMs; fewer rows use the CUDA-core matvec.
 * Default 8 (at 7B, 8 rows take 14.4 ms through the persistent kernel and ~7 ms
 * through the tensor-core pass); 0 keeps every pass on the matvec; otherwise 2..128. */
int dllm_ctx_set_tensor_core_rows(dllm_ctx* ctx, int min_rows);

/* ---- buffers (kernels.js:181-211) ----------------------------------------- */
/* ctx.loadWeightBits(u32arr, label) (kernels.js:181-186): one u32 per bf16
 * element holding the raw bits in its low half (weights.js:144-150). Stored on
 * the device as 2-byte bf16. Throws on empty input like the reference. */
int dllm_load_weight_bits(dllm_ctx* ctx, const uint32_t* bits, size_t n, const char* label, dllm_buf** out);
/* Same, from packed 2-byte bf16 (the safetensors byte layout). */
int dllm_load_weight_bf16(dllm_ctx* ctx, const uint16_t* bf16, size_t n, const char* label, dllm_buf** out);
/* ctx.createF32(numFloats, label) (kernels.js:188-191). Zero-filled. */
int dllm_create_f32(dllm_ctx* ctx, size_t n, const char* label, dllm_buf** out);
/* ctx.writeF32(buf, f32) (kernels.js:193). */
int dllm_write_f32(dllm_ctx* ctx, dllm_buf* buf, const float* src, size_t n);
/* ctx.readF32(buf, numFloats, label) (kernels.js:195-211): bounded blocking read. */
int dllm_read_f32(dllm_ctx* ctx, const dllm_buf* buf, float* dst, size_t n, const char* label);
/* Raw bf16 read-back of a weight buffer (test hook for the weight layout). */
int dllm_read_bf16(dllm_ctx* ctx, const dllm_buf* buf, uint16_t* dst, size_t n);
void dllm_buf_free(dllm_buf* buf);
size_t dllm_buf_bytes(const dllm_buf* buf);
void* dllm_buf_device_ptr(const dllm_buf* buf);
/* Synthetic weights generated on the device: N(0, std) rounded to bf16, from a
 * counter-based hash of (seed, element). Not on the decode path. */
int dllm_fill_normal_bf16(dllm_ctx* ctx, dllm_buf* buf, uint64_t seed, float std);
int dllm_fill_const_bf16(dllm_ctx* ctx, dllm_buf* buf, float value);
int dllm_create_bf16(dllm_ctx* ctx, size_t n, const char* label, dllm_buf** out);

/* Integer buffers: token ids, positions, offsets and mask words of the calls below. */
int dllm_create_i32(dllm_ctx* ctx, size_t n, const char* label, dllm_buf** out);
int dllm_write_i32(dllm_ctx* ctx, dllm_buf* buf, const int32_t* src, size_t n);
int dllm_read_i32(dllm_ctx* ctx, const dllm_buf* buf, int32_t* dst, size_t n);

/* ---- ops: one launcher per shader (kernels.js:222-301) --------------------- */
/* ctx.matmul(x, w, n, din, dout) (kernels.js:222-231): out[t,j] = sum_k x[t,k]*W[j,k]. */
int dllm_matmul(dllm_ctx* ctx, const dllm_buf* x, const dllm_buf* w, int n, int din, int dout, dllm_buf** out);
/* ctx.rmsnorm(x, g, n) (kernels.js:233-241): rows of hidden_size. */
int dllm_rmsnorm(dllm_ctx* ctx, const dllm_buf* x, const dllm_buf* g, int n, dllm_buf** out);
/* ctx.ropeQ / ctx.ropeK (kernels.js:243-254): in place, rotate-half pairs. */
int dllm_rope_q(dllm_ctx* ctx, dllm_buf* x, int pos_start, int n);
int dllm_rope_k(dllm_ctx* ctx, dllm_buf* x, int pos_start, int n);
/* ctx.attention(q, kCache, vCache, T0, n) (kernels.js:256-268): causal GQA over
 * fp32 caches laid out [max_pos, KVH*HD] as Stage.kv holds them (pipeline.js:38-43). */
int dllm_attention(dllm_ctx* ctx, const dllm_buf* q, const dllm_buf* kcache, const dllm_buf* vcache, int t0, int n,
                   dllm_buf** out);
/* ctx.siluMul(a, b, total) (kernels.js:270-279). */
int dllm_silu_mul(dllm_ctx* ctx, const dllm_buf* a, const dllm_buf* b, int total, dllm_buf** out);
/* ctx.add(a, b, n) (kernels.js:281-289); bounds-checked, unlike the shader. */
int dllm_add(dllm_ctx* ctx, const dllm_buf* a, const dllm_buf* b, int n, dllm_buf** out);
/* ctx.addBias(a, bias, n, dout) (kernels.js:291-301). */
int dllm_add_bias(dllm_ctx* ctx, const dllm_buf* a, const dllm_buf* bias, int n, int dout, dllm_buf** out);
/* Greedy argmax over n fp32 logits with the host scan's rule (pipeline.js:159-162):
 * strict '>' in index order, so the lowest index wins ties; NaN never wins. */
int dllm_argmax(dllm_ctx* ctx, const dllm_buf* logits, int n, int32_t* index_out);

/* ---- Stage: contiguous layer range + KV cache (pipeline.js:26-88) ---------- */
int dllm_stage_create(dllm_ctx* ctx, int start, int end, dllm_stage** out);  /* new Stage(k, start, end) */
void dllm_stage_destroy(dllm_stage* st);
/* stage.W[name] = buf (pipeline.js:31). HF tensor names (weights.js:167-182). */
int dllm_stage_set_weight(dllm_stage* st, const char* name, dllm_buf* buf);
/* Stage.reset() (pipeline.js:37-46): T0 = 0 for every sequence. */
int dllm_stage_reset(dllm_stage* st);
/* Stage.T0 for sequence `seq` (pipeline.js:33). */
int dllm_stage_get_t0(const dllm_stage* st, int seq);
int dllm_stage_set_t0(dllm_stage* st, int seq, int t0);
/* Stage.forward(hiddenF32, n, posStart) (pipeline.js:48-78) on sequence 0:
 * uploads n rows, runs the layers, T0 += n, returns the new hidden buffer. */
int dllm_stage_forward(dllm_stage* st, const float* hidden, int n, int pos_start, dllm_buf** out);
/* Device-resident decode pass of one micro-batch (the stage side of a hop,
 * script.js:163-172, with the hidden rows already in device memory): row i of
 * `h_dev` ([m, D] fp32, 1 <= m <= 8) belongs to sequence seq_ids[i] (host
 * array, distinct) at position == slot == that sequence's T0; h is updated in
 * place and every listed sequence's T0 advances by one. Optional device arrays:
 * tokens_in_dev[m] first replaces h with the token embeddings (embedTokens,
 * pipeline.js:121-128; needs model.embed_tokens.weight); tokens_out_dev[m]
 * receives the greedy tokens of final norm + LM head (sampleLast,
 * pipeline.js:141-174; needs model.norm.weight and a LM head). */
int dllm_stage_forward_rows(dllm_stage* st, float* h_dev, int m, const int32_t* seq_ids, const int32_t* tokens_in_dev,
                            int32_t* tokens_out_dev);
/* Stage.appendKv(L, kk, vv, n) (pipeline.js:80-87): rows -> slots T0..T0+n-1. */
int dllm_stage_append_kv(dllm_stage* st, int layer, const dllm_buf* kk, const dllm_buf* vv, int n);
/* Reads KV slots back in the reference layout [n_slots, KVH*HD] fp32
 * (which: 0 = k, 1 = v). Test hook for slot indexing. */
int dllm_stage_read_kv(dllm_stage* st, int layer, int which, int seq, int slot_start, int n_slots, float* dst);
/* Synthetic prefilled KV: slots [0, n_slots) of `seq` in every layer get N(0,1)
 * values from a counter-based hash; T0 = position = n_slots. */
int dllm_stage_fill_kv_random(dllm_stage* st, int seq, int n_slots, uint64_t seed);
/* Replace the logical->physical page map of one sequence (pages must be
 * distinct and < max_seqs * pages_per_seq). Test hook for the paged layout. */
int dllm_stage_set_page_table(dllm_stage* st, int seq, const int32_t* pages, int n_pages);
int dllm_stage_pages_per_seq(const dllm_stage* st);
/* Reads the latest pass's per-row workspace of the stage's last layer: which 0 =
 * q after bias and RoPE [rows, NQ*HD] (the input of ctx.attention,
 * pipeline.js:62-65), 1 = attention output [rows, NQ*HD] (pipeline.js:65),
 * 2 = SiLU(gate)*up [rows, I] (pipeline.js:72). Test hook for op-level checks of
 * the fused phases (the reference creates one buffer per op, kernels.js:222-301). */
int dllm_stage_read_workspace(dllm_stage* st, int which, int rows, float* dst);
/* Tracing (the reference logs performance.now() deltas, pipeline.js:144,158,172):
 * with cap > 0 every stage-kernel launch stamps the GPU global timer (ns) at
 * its start and after each grid barrier into a device buffer of `cap` entries
 * (0 turns it off). Per decode pass: start, [embed], then 5 per layer (after
 * QKV, attention, O, gate/up, down), then [head]. Reads the latest launch's. */
int dllm_stage_set_trace(dllm_stage* st, int cap);
int dllm_stage_read_trace(dllm_stage* st, uint64_t* out, int cap);

/* ---- LeaderPipeline (pipeline.js:91-282), local stage only ------------------ */
/* new LeaderPipeline(k, [start,end), ...) (pipeline.js:92-107). */
int dllm_leader_create(dllm_ctx* ctx, int start, int end, dllm_leader** out);
void dllm_leader_destroy(dllm_leader* ld);
/* The leader's own Stage (pipeline.js:95), borrowed. */
dllm_stage* dllm_leader_stage(dllm_leader* ld);
/* loadLeaderWeights(embedBits, normBits) (pipeline.js:109-119) plus the untied
 * `lm_head.weight` used by 7B/32B (NULL when tied). Buffers are referenced. */
int dllm_leader_set_weights(dllm_leader* ld, dllm_buf* embed, dllm_buf* norm, dllm_buf* lm_head);
/* embedTokens(tokens) (pipeline.js:121-128): host f32 [n, D]. */
int dllm_leader_embed_tokens(dllm_leader* ld, const int32_t* tokens, int n, float* out);
/* sampleLast(hidden) (pipeline.js:141-174): final RMSNorm, LM head, greedy
 * argmax (lowest index wins ties). `logits_out` (host, vocab floats) may be NULL. */
int dllm_leader_sample_last(dllm_leader* ld, const float* hidden_row, int32_t* token, float* logits_out);
/* forward(hidden, n, posStart) (pipeline.js:187-224) through the local stage;
 * writes the last row (D floats) to `last_row`. */
int dllm_leader_forward(dllm_leader* ld, const float* hidden, int n, int pos_start, float* last_row);
/* generate(tokens, maxNew) (pipeline.js:255-281): prefill, then greedy decode
 * with the EOS break; one CUDA-graph replay per token with the token read back
 * to the host every step. Emitted ids go to `out` (capacity max_new). */
int dllm_leader_generate(dllm_leader* ld, const int32_t* tokens, int n_tokens, int max_new, int32_t* out, int* n_out);
/* Device-resident decode: `steps` greedy tokens after `first_token` at the
 * current T0 (position == slot == T0), no EOS break and no per-step host round
 * trip (one CUDA-graph replay per token). Same token loop as generate's decode
 * branch (pipeline.js:262-267). */
int dllm_leader_decode(dllm_leader* ld, int32_t first_token, int steps, int32_t* out);
/* The same, split: enqueue the replays on the ctx stream without waiting, then
 * read the emitted tokens (bounded wait). */
int dllm_leader_decode_enqueue(dllm_leader* ld, int32_t first_token, int steps);
int dllm_leader_read_tokens(dllm_leader* ld, int32_t* out, int steps);
/* Keep the logits of the first `keep` steps of each generate/decode call in
 * device memory (0 = off, the default). */
int dllm_leader_set_keep_logits(dllm_leader* ld, int keep);
/* Logits of the most recent sampleLast, or of the last kept generate/decode step. */
int dllm_leader_last_logits(dllm_leader* ld, float* out);
/* Logits of kept step `index` (0 = the prefill's sample) of the latest call. */
int dllm_leader_read_logits(dllm_leader* ld, int index, float* out);

/* ---- multi-GPU pipeline (pipeline.js:6-87 layer-range stages, :91-282 leader loop) ----
 * One process (or thread) per GPU holds one Stage of a contiguous layer range
 * (assignLayers, pipeline.js:6-23); rank 0's stage also embeds tokens, the last
 * rank's stage holds the final norm and LM head. n_micro micro-batches of
 * `micro` sequences (sequence ids b*micro .. (b+1)*micro-1 of every stage's KV
 * cache) circulate the ring rank 0 -> 1 -> ... -> last -> 0, so with n_micro >=
 * world every GPU works on some micro-batch at once. The hidden-row hop of the
 * reference (frames over WebRTC, pipeline.js:226-253) is fused into the stage
 * kernel: a pass ends by storing its rows (the last stage: its greedy tokens) in
 * the next GPU's receive buffer over NVLink and releasing a flag there; the next
 * pass starts with a bounded wait on its flag. No host round trip per hop.
 * Set-up: every rank creates its pipeline, publishes dllm_pipeline_handle
 * (a CUDA IPC handle of its receive buffer) over the host's own channel, and
 * connects to the handle of rank (rank + 1) % world. Before the first run all
 * ranks should be connected (a host barrier), since a pass waits for its input
 * at most a few seconds. */
typedef struct dllm_pipeline dllm_pipeline;
#define DLLM_PIPELINE_HANDLE_BYTES 64
/* micro <= 8; n_micro * micro <= the stage's max_seqs. Row i of micro-batch b is
 * sequence b*micro + i at its current T0 (position == slot == T0). */
int dllm_pipeline_create(dllm_stage* st, int rank, int world, int n_micro, int micro, dllm_pipeline** out);
void dllm_pipeline_destroy(dllm_pipeline* pl);
/* This rank's receive buffer as DLLM_PIPELINE_HANDLE_BYTES opaque bytes. */
int dllm_pipeline_handle(const dllm_pipeline* pl, uint8_t* handle_out);
/* Map the receive buffer of rank (rank + 1) % world (its dllm_pipeline_handle). */
int dllm_pipeline_connect(dllm_pipeline* pl, const uint8_t* next_rank_handle);
/* Rank 0: the first token of every sequence (n_micro * micro, in sequence order). */
int dllm_pipeline_set_tokens(dllm_pipeline* pl, const int32_t* tokens, int n);
/* Enqueue `steps` greedy decode steps of every micro-batch (steps * n_micro
 * passes on this rank, in ring order) on the stage ctx's stream; no host wait. */
int dllm_pipeline_run(dllm_pipeline* pl, int steps);
/* Last rank: the tokens sampled by the latest run, [steps][n_micro * micro]
 * (bounded wait; a pass whose input never arrived reports DLLM_ETIMEOUT). */
int dllm_pipeline_read_tokens(dllm_pipeline* pl, int32_t* out, int steps);
/* Bounded wait for this rank's enqueued passes, then its device error flag. */
int dllm_pipeline_synchronize(dllm_pipeline* pl, int timeout_ms);
/* Host-fed token loop (the reference's leader: sampled tokens come back to the
 * host, pipeline.js:262-267): with `on`, the last stage keeps its tokens and the
 * first stage takes each micro-batch's tokens from dllm_pipeline_run_micro. All
 * ranks switch together, between passes. */
int dllm_pipeline_set_host_tokens(dllm_pipeline* pl, int on);
/* One pass of micro-batch b on this rank. First stage (host-token mode):
 * `tokens` (host, micro ids) are copied in first. Last stage: the sampled tokens
 * are copied to `tokens_out` (host) with a bounded wait. Others: enqueued only. */
int dllm_pipeline_run_micro(dllm_pipeline* pl, int b, const int32_t* tokens, int32_t* tokens_out);

/* ---- attention that allocates nothing ---------------------------------------
 * No counterpart in the reference. For callers that must not allocate device
 * memory: a host that owns the whole HBM budget through its own pool and forbids
 * allocations after start-up, or a latency-critical loop that cannot afford
 * cudaMalloc/cudaFree (which may synchronise the device). Same math as
 * dllm_attention (kernels.js:86-132 semantics; caches [max_pos, KVH*HD] fp32,
 * row t attends slots [0, t0+t]), but the caller passes every buffer as a device
 * pointer and the split partials, ticket counters, row descriptors and error word
 * live in a 4 MiB static device array that every GPU loading this library holds
 * until the process exits. No ctx is needed; work is enqueued on `cuda_stream`
 * (NULL: the legacy default stream) and the call does not wait for it.
 * Each call, with the caller's device current, resolves the array's device address
 * and sets the kernel's shared-memory limit (cheap, allocation-free, nothing cached,
 * so a device reset between calls is harmless). Calls share the array: calls that
 * overlap on the GPU (other streams, other threads) race. Limits: 1 <= n <= 64 rows
 * (DLLM_ERANGE beyond), head_dim 64 or 128, at most 8 query heads per KV head
 * (DLLM_EINVAL otherwise).
 * The return value covers the arguments and the launch only. Errors the kernels
 * find on the device (a split-merge wait that ran out, a row outside the cache)
 * are read with dllm_attention_noalloc_status after the call and before the next
 * one (the next call clears them). */
int dllm_attention_noalloc(const float* q, const float* kcache, const float* vcache, float* out, int t0, int n,
                           int num_q_heads, int num_kv_heads, int head_dim, int max_pos, void* cuda_stream);
/* Waits (bounded by timeout_ms, <= 0: 15000) for `cuda_stream`, then reads the
 * device error word of the latest dllm_attention_noalloc on the current device.
 * Returns DLLM_OK when the kernels reported nothing, DLLM_ETIMEOUT when a split
 * merge gave up waiting (or the stream wait itself timed out), DLLM_ERANGE when a
 * row fell outside the cache, DLLM_EDEVICE for other device codes; the raw device
 * code goes to *device_error (may be NULL). Allocates nothing. No counterpart in
 * the reference (readF32's bounded wait, kernels.js:201-207, is the model). */
int dllm_attention_noalloc_status(void* cuda_stream, int timeout_ms, int* device_error);

/* ---- verification of drafted tokens --------------------------------------------
 * No counterpart in the reference, which decodes one token per pass. A draft
 * proposes a tree of tokens per sequence; one pass scores all nodes, and a path
 * that the model agrees with is kept:
 *   dllm_tree_create         the trees' shape
 *   dllm_rope_at             q and k at the nodes' positions, T0 + depth
 *   dllm_stage_append_tree   K/V rows of the nodes, behind the cached context
 *   dllm_stage_tree_attention  every node over the context and its own ancestors
 *   dllm_pick_tokens         one token per node under penalties, biases and a mask
 *   dllm_stage_commit_tree   keep a path's K/V rows, T0 += its length
 * dllm_stage_forward_tree is the whole pass for a stage's layers: projections, the
 * config's rotary positions (as in dllm_stage_forward: whole heads, half layout, no
 * scaling), the nodes' K/V rows and their attention. The parts serve hosts with layers
 * of their own, dllm_rope_at those with other rotary positions. All work is enqueued on the ctx stream, in order; scratch
 * belongs to the ctx, so calls of one ctx, and graphs captured from them, must not
 * overlap on the GPU. T0 values become kernel arguments: a captured call replays with
 * those of its capture, and refers to the buffers, trees and plans it was given. Refused
 * while the ctx stream is captured: dllm_tree_create, dllm_rope_plan_create,
 * dllm_stage_commit_tree, dllm_stage_forward_tree, dllm_write_i32, dllm_read_i32 and
 * dllm_read_f32. A captured dllm_write_f32 reads its source with every replay, and
 * buffers are to be made before a capture. */

typedef struct dllm_tree dllm_tree;
typedef struct dllm_rope_plan dllm_rope_plan;

enum { DLLM_ROPE_HALF = 0, DLLM_ROPE_INTERLEAVED = 1 };
enum { DLLM_ROPE_PLAIN = 0, DLLM_ROPE_LINEAR = 1, DLLM_ROPE_NTK = 2, DLLM_ROPE_YARN = 3 };
typedef struct dllm_rope_config {
  int32_t layout;            /* pairs (i, i + rotary_dim / 2), or (2i, 2i + 1) */
  int32_t rotary_dim;        /* leading dims of a head that turn: even, 2..head_dim */
  double theta;              /* inverse frequency i: theta^(-2i / rotary_dim) */
  int32_t scaling;           /* PLAIN; LINEAR: frequencies / factor; NTK: theta * factor^(rd / (rd - 2));
                                YARN: a ramp from plain (fast pairs) to linear (slow pairs) */
  double factor;             /* >= 1 (not PLAIN) */
  int32_t original_max_pos;  /* YARN: the context the frequencies were trained on */
  double beta_fast, beta_slow; /* YARN: turns over that context between which the ramp runs (32, 1) */
  double attention_factor;   /* scales cos and sin; 0: 0.1 ln(factor) + 1 for YARN, else 1 */
} dllm_rope_config;
int dllm_rope_plan_create(dllm_ctx* ctx, const dllm_rope_config* cfg, dllm_rope_plan** out);
void dllm_rope_plan_destroy(dllm_rope_plan* plan);
/* Row t of q [n, NQ*HD] and k [n, KVH*HD] (either may be NULL) at positions[t] (i32,
 * any value); q_out / k_out NULL: in place. Angles are reduced in 64 bits, so
 * positions far beyond 2^24 keep their precision (dllm_rope_q/k multiply in 32). */
int dllm_rope_at(dllm_ctx* ctx, const dllm_rope_plan* plan, const dllm_buf* positions, int n, dllm_buf* q, dllm_buf* k,
                 dllm_buf* q_out, dllm_buf* k_out);

/* Trees of n_seqs sequences (1..128): counts[i] nodes (0..64) for cache sequence
 * seqs[i] (NULL: i; distinct), their parents in turn: an index within the sequence
 * below the node's own, or -1 for a root. Node j of a sequence is batch row (nodes
 * of the sequences before) + j, and its K/V row goes to slot T0 + j. */
int dllm_tree_create(dllm_ctx* ctx, const int32_t* parents, const int32_t* counts, const int32_t* seqs, int n_seqs,
                     dllm_tree** out);
void dllm_tree_destroy(dllm_tree* tree);

/* Arguments of dllm_pick_tokens; optional buffers may be NULL. V = vocab_size; the
 * sequences are the tree's, or without a tree the n rows themselves. */
typedef struct dllm_pick {
  int32_t n;                       /* 1..8192 */
  const dllm_buf* logits;          /* f32 [n, V] */
  const dllm_buf* history;         /* i32: tokens of all sequences; ids outside [0, V) are ignored */
  const dllm_buf* history_offsets; /* i32 [seqs + 1]: sequence s has [offsets[s], offsets[s + 1]) */
  const dllm_buf* prompt_lens;     /* i32 [seqs]: leading tokens that were given, not generated; NULL: none. Beyond
                                      the history they are the first tokens of a node's path */
  const dllm_buf* penalties;       /* f32 [seqs, 3]: repetition, frequency, presence */
  const dllm_buf* bias_tokens;     /* i32: entries of all sequences; of a token listed twice the last one counts */
  const dllm_buf* bias_values;     /* f32 */
  const dllm_buf* bias_offsets;    /* i32 [seqs + 1] */
  const dllm_buf* mask;            /* i32 [n, ceil(V / 32)]: bit t % 32 of word t / 32 allows token t */
  const dllm_tree* tree;           /* rows are the tree's nodes */
  const dllm_buf* draft;           /* i32 [n], with a tree: the nodes' tokens */
  dllm_buf* out;                   /* f32 [n, V]: the processed logits; may be `logits` */
  dllm_buf* tokens;                /* i32 [n]; may be `draft`, no other input */
} dllm_pick;
/* With c = occurrences of token t among the generated tokens of the row's history (a
 * node's history ends with the drafted tokens from its root to itself, so a root that
 * is the sequence's last token is not in `history` itself):
 *   y = x > 0 ? x / repetition : x * repetition   where t occurs in the history
 *   y = y - frequency * c - presence              where c > 0
 *   y += bias; y = -inf where the mask forbids t
 * tokens[row] is the lowest allowed index with the largest y (NaN counts as -inf), or
 * -1 where the mask allows nothing. Offsets outside their buffers are clamped. */
int dllm_pick_tokens(dllm_ctx* ctx, const dllm_pick* args);

/* K/V rows k, v [n, KVH*HD] fp32 -> slots T0 + node of each sequence; T0 unchanged. */
int dllm_stage_append_tree(dllm_stage* st, int layer, const dllm_tree* tree, const dllm_buf* k, const dllm_buf* v);
/* out[row] = attention of node `row` (q [n, NQ*HD], after RoPE) over its sequence's
 * slots [0, T0) and the slots of its ancestors and itself. A non-finite value in a
 * drafted K/V row reaches only the nodes that see the row; there, an infinity may come
 * out as NaN. */
int dllm_stage_tree_attention(dllm_stage* st, int layer, const dllm_tree* tree, const dllm_buf* q, dllm_buf* out);
/* Keep one path per sequence: lens[i] node indices (a root, then a child each; 0: keep
 * nothing), all sequences' in turn in `path`. Slot T0 + path[j] -> T0 + j in every
 * layer of the stage; T0 += lens[i]. The slots behind hold leftovers. */
int dllm_stage_commit_tree(dllm_stage* st, const dllm_tree* tree, const int32_t* path, const int32_t* lens);
/* Every layer of the stage for the tree's rows (at most 128): h [n, D] in place; `tokens`
 * (i32 [n], may be NULL) first replaces h by their embeddings; `logits` (f32 [n, V], may
 * be NULL) receives final norm + LM head. K/V rows are appended, T0 is unchanged. */
int dllm_stage_forward_tree(dllm_stage* st, const dllm_tree* tree, dllm_buf* h, const dllm_buf* tokens,
                            dllm_buf* logits);
/* The stage's K (which = 0) or V (1) pool on the device, [layers][max_seqs *
 * pages_per_seq][KVH][page][HD] in the cache's type, for hosts that fill or inspect the
 * cache with kernels of their own on the ctx stream. */
void* dllm_stage_kv_device_ptr(const dllm_stage* st, int which);

/* ---- long conversations -----------------------------------------------------------
 * No counterpart in the reference. For hosts with layers of their own: norms of the query
 * and key heads, K/V rows of a batch, attention under a sliding window and first tokens
 * that stay visible ("sinks"), and a cache that holds K and V in 4 bits.
 * A batch of rows (dllm_rows) says how many rows each of its sequences has: one new token,
 * a chunk of a prompt, or none. Row j of a sequence is cache slot T0 + j. As with drafted
 * trees, work is enqueued on the ctx stream in order, scratch belongs to the ctx (calls of
 * one ctx, and graphs captured from them, must not overlap on the GPU), and T0 values are
 * those of the call: a captured call replays with them, and refers to the buffers it was
 * given. dllm_rows_create, dllm_kv4_create, dllm_kv4_set_page_table are refused while the
 * ctx stream is captured, and so is attention of a long chunk that needs more scratch than
 * any call before: make the call once outside. (Scratch is 2 bytes per K or V value that long
 * chunks see in a bf16 cache, 4 in the others, up to 1 GB or one sequence's share.) */

/* For every head of q [n, NQ*HD] and k [n, KVH*HD] (either may be NULL, with its norm):
 * y = x / sqrt(mean(x^2) + rms_norm_eps) * norm, norm a bf16 weight [HD]; then the plan's
 * rotation at positions[t], as in dllm_rope_at. q_out / k_out NULL: in place. */
int dllm_norm_rope_at(dllm_ctx* ctx, const dllm_rope_plan* plan, const dllm_buf* positions, int n, dllm_buf* q, dllm_buf* k,
                      const dllm_buf* q_norm, const dllm_buf* k_norm, dllm_buf* q_out, dllm_buf* k_out);

/* counts[i] rows (0..max_pos) for cache sequence seqs[i] (NULL: i; distinct), 1..128
 * sequences and 1..1048576 rows in all. */
typedef struct dllm_rows dllm_rows;
int dllm_rows_create(dllm_ctx* ctx, const int32_t* counts, const int32_t* seqs, int n_seqs, dllm_rows** out);
void dllm_rows_destroy(dllm_rows* rows);

/* K/V rows k, v [n, KVH*HD] fp32 -> slots T0 + j of each sequence; T0 unchanged. */
int dllm_stage_append_rows(dllm_stage* st, int layer, const dllm_rows* rows, const dllm_buf* k, const dllm_buf* v);
/* out[row] = attention of the row at slot p = T0 + j (q [n, NQ*HD], after RoPE) over its
 * sequence's slots s <= p with s > p - window or s < sinks; window 0: all of them. The rows'
 * own K/V are in the cache before. Fp32 arithmetic: products keep 22 bits of q, of p, and of the largest
 * fp32 value of each K or V row. A K/V value reaches only the rows that see it, whatever its size (an
 * infinity may come out as NaN there). */
int dllm_stage_window_attention(dllm_stage* st, int layer, const dllm_rows* rows, const dllm_buf* q, dllm_buf* out,
                                int window, int sinks);

/* A cache of layers [start, end) in 4 bits: max_seqs sequences of max_pos slots in pages of
 * kv_page_size, as a stage has them, and T0 per sequence. Each 32 dims of a K or V row
 * share a minimum m and a scale s in bf16 (5 bits per value in all): a value is m + c s,
 *   m = the smallest of the 32 rounded down, s = fp32((largest - m) / 15) rounded up,
 *   c = (x - m) / s to the nearest of 0..15 (ties to even)
 * so that it is off by s / 2 at most. 32 values with a NaN, a number beyond bf16's largest (3.39e38;
 * infinities are) or a range of 2^112 and more among them all read NaN. */
typedef struct dllm_kv4 dllm_kv4;
int dllm_kv4_create(dllm_ctx* ctx, int start, int end, dllm_kv4** out);
void dllm_kv4_destroy(dllm_kv4* kv);
int dllm_kv4_reset(dllm_kv4* kv);
int dllm_kv4_get_t0(const dllm_kv4* kv, int seq);
int dllm_kv4_set_t0(dllm_kv4* kv, int seq, int t0);
int dllm_kv4_pages_per_seq(const dllm_kv4* kv);
int dllm_kv4_set_page_table(dllm_kv4* kv, int seq, const int32_t* pages, int n_pages);
/* Device memory of the cache (codes, scales and minima). */
size_t dllm_kv4_bytes(const dllm_kv4* kv);
/* K/V rows k, v [n, KVH*HD] fp32 -> slots T0 + j of each sequence; T0 unchanged. */
int dllm_kv4_append(dllm_kv4* kv, int layer, const dllm_rows* rows, const dllm_buf* k, const dllm_buf* v);
/* The values that slots T0 + j stand for, fp32 [n, KVH*HD]; either output may be NULL. */
int dllm_kv4_read_rows(dllm_kv4* kv, int layer, const dllm_rows* rows, dllm_buf* k, dllm_buf* v);
/* dllm_stage_window_attention over this cache's values. */
int dllm_kv4_attention(dllm_kv4* kv, int layer, const dllm_rows* rows, const dllm_buf* q, dllm_buf* out, int window,
                       int sinks);

#ifdef __cplusplus
}
#endif
#endif /* DLLM_H */
