/* llmq_cuda.h - C ABI of libllmq_cuda.so, the B200 (sm_100a) implementation of the
 * int8 (W8A8) LLaMA-family KV-cache decode path of marjoncajocon/llm-project.
 *
 * The library is a link-time drop-in for the int8 half of the reference:
 *   quant.c in full (quant.h:15-33) and the QLlamaModel section of llama.c
 *   (llama.c:443-657, declared at llama.h:114-140) plus llama_kv_free (llama.h:102).
 * Every exported name, argument order, struct layout, ownership rule and return
 * convention below is the reference's, so a caller written against quant.h /
 * llama.h compiles and links unchanged.  All arithmetic runs on the GPU: the
 * results are bit-identical to the reference CPU code (same int8 codes, same
 * int32 accumulators, same fp32 rounding sequence, the same libm expf results).
 *
 * Additions (new names, same C style) carry a comment saying so.  No entry point
 * takes or returns a torch or CUDA type.  Compute functions that return void in the
 * reference keep returning void; their failures are reported by
 * q_llama_last_error() and a one-line message on stderr.
 */
#ifndef LLMQ_CUDA_H
#define LLMQ_CUDA_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* ------------------------------------------------------------------------- */
/* Host structs.  The guards are the reference headers' own include guards, so */
/* this header and tensor.h / quant.h / llama.h may be included in any order.  */
/* ------------------------------------------------------------------------- */
#ifndef TENSOR_H
#define TENSOR_H
/* Same layout as the reference Tensor (tensor.h:10-16): row-major f32 data,
 * optional grad, malloc'd shape array.  Tensors this library allocates use a
 * 64-byte aligned `data` block and a malloc'd `shape`, like tensor.c:33-60, so
 * the reference tensor_free can release them. */
typedef struct {
  float *data;
  float *grad;
  int *shape;
  int ndim;
  size_t size;
} Tensor;
#endif

#ifndef QUANT_H
#define QUANT_H
/* int8 weight, (rows=in, cols=out) row-major, one f32 scale per column
 * (quant.h:22-26).  x(M,rows) @ W -> (M,cols). */
typedef struct {
  int rows, cols;
  signed char *q;
  float *scale;
} QTensor;
#endif

#ifndef LLAMA_H
#define LLAMA_H
/* fp32 block / model (llama.h:19-36, 59-66).  Only read here, by
 * q_llama_quantize_from. */
typedef struct {
  int d_model, n_heads, n_kv, head_dim, d_ff;
  float rope_base, eps;
  Tensor attn_norm, Wq, Wk, Wv, b_q, b_k, b_v, Wo;
  Tensor ffn_norm, Wgate, Wup, Wdown;
} LlamaBlock;

typedef struct {
  int vocab, d_model, n_layers, n_heads, n_kv, head_dim, d_ff, max_seq;
  float rope_base, eps;
  Tensor wte;
  LlamaBlock *blocks;
  Tensor final_norm;
  Tensor lm_head;
} LlamaModel;

/* KV cache handle (llama.h:94-99).  `len` is the number of cached positions and
 * is the source of truth on every call: callers restart a sequence by writing
 * kv.len = 0 (main.c:661).  The cache itself lives on the GPU; the host arrays
 * k/v are allocated with the reference's shapes and are filled only by
 * q_llama_kv_sync_host(). */
typedef struct {
  int n_layers, max_seq, kv_dim;
  int len;
  float **k;
  float **v;
} LlamaKV;

/* int8 block / model (llama.h:114-127). */
typedef struct {
  Tensor attn_norm, ffn_norm;
  Tensor b_q, b_k, b_v;
  QTensor Wq, Wk, Wv, Wo, Wgate, Wup, Wdown;
} QLlamaBlock;

typedef struct {
  int vocab, d_model, n_layers, n_heads, n_kv, head_dim, d_ff, max_seq;
  float rope_base, eps;
  QTensor wte;
  QLlamaBlock *blocks;
  Tensor final_norm;
  QTensor lm_head;
} QLlamaModel;
#endif

#ifndef SAMPLER_H
#define SAMPLER_H
/* xorshift64 stream (sampler.h:13-15). */
typedef struct {
  unsigned long long state;
} Rng;
#endif

/* ========================================================================= */
/* quant.h entry points                                                       */
/* ========================================================================= */

/* Replaces quant.c:10-27 (declared quant.h:15).  Per-column symmetric int8
 * quantisation of a row-major (rows, cols) f32 matrix, computed on the GPU:
 * scale[j] = max_i|w[i,j]|/127 (1 for an all-zero column),
 * q = clamp(lrintf(w * (1/scale[j])), -127, 127).  Bit-identical to the
 * reference.  Host pointers in and out. */
void quantize_int8_percol(const float *w, int rows, int cols, signed char *q, float *scale);

/* Replaces quant.c:29-33 (quant.h:16).  w[i,j] = q[i,j] * scale[j], on the GPU. */
void dequantize_int8_percol(const signed char *q, const float *scale, int rows, int cols, float *w);

/* Replace quant.c:35-50 (quant.h:28-30).  Host allocation, as in the reference. */
QTensor qtensor_create(int rows, int cols);
void qtensor_free(QTensor *t);
void qtensor_quantize(QTensor *t, const float *w);

/* Replaces quant.c:60-85 (quant.h:33).  C(M,N) = W8A8 product of A(M,K) with W:
 * each row of A is quantised to int8 with its own absmax scale, multiplied
 * exactly in int32 against W's codes, and rescaled as a_scale*w_scale[j]*acc.
 * A, W and C are host memory, read and written on every call exactly like the
 * reference: each call copies A and W to the GPU (W is tiled there) and C back,
 * so a QTensor rewritten in place between calls is always seen. */
void qmatmul(const Tensor *A, const QTensor *W, Tensor *C);

/* ========================================================================= */
/* llama.h entry points (int8 model)                                          */
/* ========================================================================= */

/* Replaces llama.c:610-657 (llama.h:136).  Reads an LLMQ v2 checkpoint into
 * host memory exactly like the reference (0 on success, 1 with a message on
 * stderr on any error; the model is freed on failure) and uploads it to the
 * current GPU.  With a tensor-parallel group formed (q_llama_tp_init) it only
 * reads: the whole model is then meant to be cut with q_llama_model_shard. */
int q_llama_model_load(const char *path, QLlamaModel *out);

/* Replaces llama.c:483-488 (llama.h:129).  Frees host arrays and the device copy
 * (weights, every KV cache and CUDA graph made for this model). */
void q_llama_model_free(QLlamaModel *m);

/* Replaces llama.c:490-511 (llama.h:132).  Quantises an fp32 model on the GPU
 * (bit-identical codes and scales). */
QLlamaModel q_llama_quantize_from(const LlamaModel *src);

/* Replaces llama.c:513-526 (llama.h:140).  Creates the GPU KV cache
 * (head-major f32 [n_layers][n_kv][max_seq][head_dim], K and V) plus the reference-shaped host
 * arrays. */
LlamaKV q_llama_kv_create(const QLlamaModel *m);

/* Replaces llama.c:290-294 (llama.h:102) for caches made by q_llama_kv_create. */
void llama_kv_free(LlamaKV *kv);

/* Replaces llama.c:528-600 (llama.h:139).  Decodes `token` at position kv->len:
 * appends its K/V to the GPU cache, attends over 0..kv->len, writes the f32
 * logits (1, vocab) into the caller's host tensor and advances kv->len.  One
 * CUDA graph replay per call. */
void q_llama_decode_step(const QLlamaModel *m, LlamaKV *kv, int token, Tensor *logits);

/* ========================================================================= */
/* llama.h fp32 (LLMA) decode entry points                                   */
/* ========================================================================= */

/* Replaces llama.c:275-288 (llama.h:101): the KV cache of an fp32 model, on
 * the GPU (head-major as for the int8 model) plus the reference-shaped host
 * arrays.  The model's GPU copy is made on first use. */
LlamaKV llama_kv_create(const LlamaModel *m);

/* Replaces llama.c:296-362 (llama.h:106): one decode step of an fp32 model on
 * the GPU, bit-identical to the reference's.  Every product is fp32 with the
 * reference's accumulation order (matrix.c:178-199: one sequential chain per
 * output column, each product and sum rounded on its own); norms, RoPE,
 * attention and SwiGLU are the int8 path's kernels.  The model is
 * snapshotted at its first use: release the GPU copy with
 * llmq_llama_model_release (or llmq_llama_model_free) before editing it. */
void llama_decode_step(const LlamaModel *m, LlamaKV *kv, int token, Tensor *logits);

/* As llama_decode_step; returns the greedy next id (-1 on error); logits may
 * be NULL.  Additive extension. */
int llama_decode_step_argmax(const LlamaModel *m, LlamaKV *kv, int token, Tensor *logits);
/* As q_llama_decode_step_sample, for an fp32 model. */
int llama_decode_step_sample(const LlamaModel *m, LlamaKV *kv, int token, float temperature, int top_k,
                             float top_p, Rng *rng, Tensor *logits);
/* As q_llama_generate / q_llama_generate_sample, for an fp32 model. */
int llama_generate(const LlamaModel *m, LlamaKV *kv, int token, int n, int *ids);
int llama_generate_sample(const LlamaModel *m, LlamaKV *kv, int token, int n, float temperature, int top_k,
                          float top_p, Rng *rng, int *ids);

/* llama.c:390-440 under a name of this library: reads an LLMA (f32) or LLMQ
 * (int8, dequantised on load as quant.c:29-33) checkpoint into an fp32 model
 * in host memory (the GPU copy is made on first use).  Same messages and 0/1
 * return as llama_model_load.  Free with llmq_llama_model_free. */
int llmq_llama_model_load(const char *path, LlamaModel *out);
/* Frees a model made by llmq_llama_model_load / llmq_synth_model_f32 and its
 * GPU copy. */
void llmq_llama_model_free(LlamaModel *m);
/* Uploads / releases the GPU copy of an fp32 model (both otherwise implicit).
 * Returns 0 or an error code. */
int llmq_llama_model_upload(const LlamaModel *m);
void llmq_llama_model_release(const LlamaModel *m);

/* ========================================================================= */
/* sampler.h entry points (sampler.c, the generation loop's token choice)     */
/* ========================================================================= */

/* Replace sampler.c:26-30 and sampler.c:41-44 (host arithmetic, same stream). */
Rng rng_create(unsigned long long seed);
float rng_uniform(Rng *r);

/* Replaces sampler.c:8-21 (sampler.h:10): the first index of the largest
 * logit of row `row`, computed on the GPU. */
int sample_argmax(const Tensor *logits, int row);

/* Replaces sampler.c:60-115 (sampler.h:25-26): temperature, top-k and top-p
 * sampling of row `row` on the GPU, advancing *rng by one draw (none when
 * temperature <= 0).  The returned id equals the reference's for every input,
 * ties included (glibc's stable qsort order: p descending, then index).  The
 * GPU keeps up to 1024 candidates: top_k must be in 1..1024 unless vocab <=
 * 1024; otherwise -1 is returned with q_llama_last_error() set and *rng
 * unchanged. */
int sample_token(const Tensor *logits, int row, float temperature, int top_k, float top_p, Rng *rng);

/* ========================================================================= */
/* Additions (no counterpart in the reference headers)                        */
/* ========================================================================= */

enum {
  LLMQ_OK = 0,
  LLMQ_ERR_ARG = 1,      /* bad shape / id / position / null pointer */
  LLMQ_ERR_CUDA = 2,     /* a CUDA runtime call failed */
  LLMQ_ERR_NO_DEVICE = 3,/* no CUDA device, or not an sm_100 part */
  LLMQ_ERR_IO = 4,       /* checkpoint read / write failure */
  LLMQ_ERR_OOM = 5,      /* host or device allocation failed */
  LLMQ_ERR_STATE = 6     /* model / cache not known to this library */
};

/* Error code of the most recent failing call on this thread (LLMQ_OK if none)
 * and its message.  q_llama_clear_error resets both. */
int q_llama_last_error(void);
const char *q_llama_last_error_message(void);
void q_llama_clear_error(void);

/* As q_llama_decode_step, but also returns the greedy next token (first index
 * of the largest logit, the rule of sampler.c:8-21) computed on the GPU.
 * `logits` may be NULL, in which case no logits are copied to the host (4 bytes
 * cross PCIe per token).  Returns -1 on error. */
int q_llama_decode_step_argmax(const QLlamaModel *m, LlamaKV *kv, int token, Tensor *logits);

/* q_llama_decode_step followed by sample_token on its logits row
 * (main.c:663-668), with the sampler run on the GPU inside the same graph:
 * returns the drawn next token (-1 on error) and advances kv->len and *rng.
 * `logits` may be NULL.  temperature <= 0 takes the greedy id and draws
 * nothing; top_k follows sample_token's limit.  Additive extension. */
int q_llama_decode_step_sample(const QLlamaModel *m, LlamaKV *kv, int token, float temperature, int top_k,
                               float top_p, Rng *rng, Tensor *logits);

/* Sampled generation chained on the GPU: as q_llama_generate, with each next
 * token drawn by the sampler (the reference's loop of q_llama_decode_step and
 * sample_token, main.c:663-668).  ids[i] is the token drawn after step i;
 * kv->len advances by n and *rng by n draws.  Returns 0 or an error code. */
int q_llama_generate_sample(const QLlamaModel *m, LlamaKV *kv, int token, int n, float temperature, int top_k,
                            float top_p, Rng *rng, int *ids);

/* Batched decode: one token for each of B sequences at once.  Sequence b feeds
 * tokens[b] at position kvs[b]->len of its own cache; row b of `logits`
 * (B x vocab floats, caller-owned) receives its logits and every kvs[b]->len
 * advances by one.  Each row equals what q_llama_decode_step (llama.c:528-600)
 * gives for that sequence alone, bit for bit; the caches must be distinct.
 * The reference has no batch entry point: this is the additive
 * `q_llama_decode_batch` extension of the C API. */
void q_llama_decode_batch(const QLlamaModel *m, LlamaKV **kvs, const int *tokens, int B, Tensor *logits);

/* As q_llama_decode_batch, but writes the B greedy ids (first maximum,
 * sampler.c:8-21) to ids[] instead of logits.  Returns 0 or an error code. */
int q_llama_decode_batch_argmax(const QLlamaModel *m, LlamaKV **kvs, const int *tokens, int B, int *ids);

/* Prefill: feeds ids[0..n) at positions kv->len .. kv->len + n - 1 in one pass
 * (the tensor-core GEMMs see n rows).  The cache then equals that of n
 * q_llama_decode_step calls, and `logits` (1 x vocab, may be NULL) receives the
 * logits of the last id, bit for bit those of the n-th step.  kv->len advances
 * by n.  Additive extension (the reference feeds prompts token by token,
 * main.c:650-671). */
void q_llama_prefill(const QLlamaModel *m, LlamaKV *kv, const int *ids, int n, Tensor *logits);

/* As q_llama_prefill; returns the greedy id after the last prompt token, or -1
 * on error. */
int q_llama_prefill_argmax(const QLlamaModel *m, LlamaKV *kv, const int *ids, int n, Tensor *logits);

/* Kernels launched by the last q_llama_decode_batch[_argmax|_sample],
 * q_llama_paged_step or q_llama_prefill[_argmax] call (diagnostic; no reference
 * counterpart). */
long long llmq_last_launches(void);

/* ---- Tensor parallelism (the `q_llama_tp_init` extension; the reference is
 * single-process).  One process per GPU: select the device with
 * q_llama_set_device, have rank 0 make an id with q_llama_tp_unique_id and
 * hand its 128 bytes to every rank, then call q_llama_tp_init on all ranks
 * (it returns once all have joined).  A model whose tensors are shard `rank`
 * of `world` (llmq_synth_model_shard, q_llama_model_shard) then decodes as
 * one: Wq/Wk/Wv/Wgate/Wup and the lm-head by columns, Wo/Wdown by rows, with
 * an NCCL max-reduce of the activation absmax and a sum-reduce of the exact
 * int32 partial products per row-parallel product, and a max-reduce of the
 * argmax key.  Logits and greedy ids equal the single-GPU ones bit for bit;
 * q_llama_decode_step returns the whole logits row on every rank, and
 * q_llama_kv_sync_host fills only this rank's KV heads.  All ranks must make
 * the same calls in the same order.  Returns 0 or an error code. */
int q_llama_tp_unique_id(unsigned char *id /* 128 bytes */);
int q_llama_tp_init(int rank, int world, const unsigned char *id);
/* Releases the group's communicator (and the decode graphs that use it). */
void q_llama_tp_shutdown(void);

/* Copies the GPU KV cache rows [0, kv->len) into kv->k / kv->v (the
 * reference-shaped host arrays).  Returns LLMQ_OK or an error code. */
int q_llama_kv_sync_host(const QLlamaModel *m, LlamaKV *kv);

/* Writes an LLMQ v2 checkpoint (the layout q_llama_model_load reads,
 * llama.c:192-220 and llama.c:603-648): atomically, through `path`.tmp and a
 * rename.  Returns 0 on success, 1 with a message on stderr on error. */
int q_llama_model_save(const char *path, const QLlamaModel *m);

/* Replaces tools/upgrade_llma.py: an LLMA v1 checkpoint (no q/k/v biases)
 * becomes v2 with three zero bias vectors per layer inserted after Wv,
 * streamed in 4 MiB pieces.  Refuses non-LLMA, already-v2, truncated and
 * overlong files with the tool's messages; 0 on success, 1 on error. */
int llmq_llma_upgrade_v1(const char *src, const char *dst);

/* Model configuration, in LLMQ header order (llama.c:241-243). */
typedef struct {
  int vocab, d_model, n_layers, n_heads, n_kv, head_dim, d_ff, max_seq;
  float rope_base, eps;
} LlmqConfig;

/* Builds a seeded synthetic int8 model in host memory (not uploaded; the first
 * q_llama_kv_create / decode call uploads it).  Every 2-D weight is drawn
 * f32 N(0, stddev) from splitmix64 + Box-Muller keyed by (seed, tensor index,
 * element index), then quantised per column by the reference rule.  Norm gains
 * are 1; biases are 0, or N(0, stddev) when `with_bias` (the Qwen2 path).
 * Multi-threaded; the result does not depend on the thread count.
 * Returns 0 or an error code. */
int llmq_synth_model(const LlmqConfig *cfg, uint64_t seed, float stddev, int with_bias,
                     QLlamaModel *out);

/* The fp32 model an LLMQ checkpoint of llmq_synth_model(cfg, seed, stddev,
 * with_bias) loads as with llama_model_load (llama.c:419-427: every 2-D
 * tensor dequantised).  Free with llmq_llama_model_free.  Returns 0 or an
 * error code. */
int llmq_synth_model_f32(const LlmqConfig *cfg, uint64_t seed, float stddev, int with_bias, LlamaModel *out);

/* Tensor-parallel shard `rank` of `world` of the same synthetic model (no
 * reference counterpart): Wq/Wk/Wv and b_q/b_k/b_v keep the columns of this
 * rank's query and KV heads, Wgate/Wup its d_ff columns, lm_head its vocab
 * columns; Wo and Wdown keep the rows of its query dims and d_ff slice.  Every
 * kept code and per-column scale equals the whole model's (row shards keep the
 * scale of the whole column).  wte and the norms are whole; the config fields
 * are the whole model's.  Needs n_heads, n_kv, d_ff and vocab divisible by
 * world.  Returns 0 or an error code. */
int llmq_synth_model_shard(const LlmqConfig *cfg, uint64_t seed, float stddev, int with_bias, int rank,
                           int world, QLlamaModel *out);

/* Shard `rank` of `world` of a quickly generated benchmark model: codes uniform
 * in [-127, 127] and per-column scales uniform in [2e-4, 1e-3), seeded per
 * element, so a shard costs only its own elements (a 70B shard in seconds).
 * Same layout and shard rules as llmq_synth_model_shard; no reference
 * counterpart.  Returns 0 or an error code. */
int llmq_synth_model_fast_shard(const LlmqConfig *cfg, uint64_t seed, int rank, int world, QLlamaModel *out);

/* The same shard cut from a whole model held in host memory (for instance one
 * read by q_llama_model_load).  `out` is freed with q_llama_model_free.
 * Returns 0 or an error code. */
int q_llama_model_shard(const QLlamaModel *m, int rank, int world, QLlamaModel *out);

/* Fills an existing QTensor with uniform codes in [-127, 127] and uniform scales
 * in [1e-3, 1e-2), seeded (the isolated matvec sweep's weights). */
void llmq_synth_qtensor(QTensor *t, uint64_t seed);

/* Addition (the writer tools/convert_llama.py:73-97 is for converted models):
 * the model llmq_synth_model (fast = 0) or llmq_synth_model_fast_shard with
 * one shard (fast = 1, stddev and with_bias ignored) builds, written straight
 * to an LLMQ v2 file tensor by tensor, so no more than one tensor is ever in
 * host memory (a 70B-shaped file needs ~1 GB of RAM, not ~70 GB).  Byte for byte
 * what q_llama_model_save writes for that model; atomic like llama.c:230-269.
 * Returns 0 or an error code. */
int llmq_synth_model_save(const LlmqConfig *cfg, uint64_t seed, float stddev, int with_bias, int fast,
                          const char *path);

/* Upload / release the device copy of a model explicitly (both are otherwise
 * implicit).  Returns 0 or an error code. */
int q_llama_model_upload(const QLlamaModel *m);

/* Selects the CUDA device that later uploads, caches and standalone calls on
 * this thread use (one process per GPU: pass the local rank).  A model keeps
 * the device it was uploaded to.  Returns 0 or an error code. */
int q_llama_set_device(int device);

/* Greedy generation chained on the GPU: feeds `token` at position kv->len, then
 * keeps feeding the argmax of each step, for n steps in total (one CUDA graph
 * replay per step, no host round trip in between).  ids[i] receives the argmax
 * after step i; kv->len advances by n.  Returns 0 or an error code. */
int q_llama_generate(const QLlamaModel *m, LlamaKV *kv, int token, int n, int *ids);

/* GPU time in milliseconds of the last q_llama_decode_step[_argmax] (one step,
 * including its small host<->device copies) or q_llama_generate (all n steps),
 * from CUDA events on the model's stream. */
float q_llama_last_step_ms(void);

/* ---- diagnostics for tests and benchmarks ---- */

/* y[i] = expf(x[i]) evaluated on the GPU by the routine the decode kernels use
 * (bit-identical to the host C library's expf).  Returns 0 or an error code. */
int llmq_expf_device(const float *x, float *y, long long n);

/* Times `iters` back-to-back launches of one kernel of an uploaded model
 * (which: 0 fused QKV, 1 Wo, 2 fused W1|W3, 3 W2, 4 lm-head GEMV, 5 attention
 * over the first KV cache at its current position) with CUDA events on the
 * model's stream.  Launch i takes block (layer + i) mod n_layers, so
 * consecutive launches stream different weights; the launches are replayed
 * from one CUDA graph with programmatic dependent launch, as inside a decode
 * step, so the host's launch rate is not timed.  *ms_per_launch receives the mean
 * launch time and *bytes_per_launch the algorithmic bytes of one launch (GEMV:
 * int8 weights + f32 scales + f32 input + f32 output; attention: the K and V
 * rows read plus q and the output).  Returns 0 or an error code. */
int llmq_bench_gemv(const QLlamaModel *m, int which, int layer, int iters, float *ms_per_launch,
                    double *bytes_per_launch);

/* Kernels launched by one decode step: per layer QKV, attention (one fused
 * launch, or two), Wo, W1|W3, W2 (+ 2 absmax exchanges under tensor
 * parallelism); then lm-head and the step's bookkeeping. */
int llmq_kernels_per_step(const QLlamaModel *m);

/* Attention launches per layer of a batch-1 step with these dimensions: 1 (the
 * fused cluster kernel) or 2 (scores, then softmax and values; chosen when the
 * fused kernel's shared memory would not fit, or LLMQ_ATTN_TWO_KERNELS=1);
 * -1 without a suitable GPU. */
int llmq_attention_launches(int n_heads, int n_kv, int head_dim, int max_seq);

/* Times `iters` device-resident products C(M, N) = A(M, K) x W on the path
 * qmatmul uses (int8 GEMV for M <= 8, tcgen05 tensor cores for larger M), with
 * W tiled once and seeded A resident in device memory.  *ms receives the mean
 * time per product.  Returns 0 or an error code. */
int llmq_bench_qmatmul(const QTensor *W, int M, int iters, float *ms);

/* Runs one decode step of `token` at kv->len outside the CUDA graph, kernel by
 * kernel with CUDA events between the launches, writes each kernel's time in
 * milliseconds to ms[0 .. min(max_n, llmq_kernels_per_step(m))) and advances
 * kv->len like a decode step.  For attributing step time to kernels; the
 * kernels do not overlap here.  Returns 0 or an error code. */
int llmq_step_profile(const QLlamaModel *m, LlamaKV *kv, int token, float *ms, int max_n);

/* RMSNorm of the row x[W->rows] with gain gamma and epsilon eps
 * (rmsnorm.c:7-21), then qmatmul of the normalised row by W (quant.c:60-85):
 * out[W->cols], host arrays, computed by the GEMV with the RMSNorm prologue that
 * QKV, W1|W3 and the lm-head use in a decode step (for tests on chosen rows).
 * Returns 0 or an error code. */
int llmq_rmsnorm_qmatmul(const float *x, const float *gamma, float eps, const QTensor *W, float *out);

/* The RMSNorm's sum of squares (rmsnorm.c:15) as the GEMV prologues form it:
 * one thread block sums a row in the loop's order and rounding, its 32
 * segments run in parallel from candidate starts around estimated partial sums
 * and linked exactly.  For each of `rows` rows of
 * n floats (host array v), sums[2r] is the block's sum and sums[2r+1] the
 * one-thread loop's (equal bit for bit), misses[r] the segments whose exact
 * start was not a candidate (summed by one thread), cycles[2r] and
 * cycles[2r+1] the SM cycles of the two.  threads: block size, a multiple of
 * 32 in 64..1024.  Returns 0 or an error code. */
int llmq_spec_sum_check(const float *v, int rows, int n, int threads, float *sums, int *misses, long long *cycles);

/* Failure detection on one GPU (no reference counterpart): runs a two-rank
 * tensor-parallel exchange whose second rank is a local region nothing writes,
 * so the peer-flag waits give up after `polls` polls.  which 0: the absmax
 * exchange kernel; 1: the row-parallel GEMV.  The kernel returns by itself;
 * *err_word receives the device error word (1 = timeout) and *ms its duration.
 * Returns LLMQ_ERR_CUDA when the error word is set (as a decode step does),
 * else 0; frees everything it allocated. */
int llmq_tp_wait_timeout_check(int which, unsigned polls, int *err_word, float *ms);

/* ---- allocation-free entry point ---- */

/* No counterpart in the reference (it has no GPU).  The qmatmul product
 * (quant.c:60-85, bit-identical results) on buffers the caller already holds on
 * the current GPU, for callers that cannot call cudaMalloc where they multiply:
 * a host framework whose own memory pool already owns the GPU's memory, a plugin
 * that must not change the application's device-memory accounting, or a
 * latency-critical loop that cannot afford an allocation and the device
 * synchronisation of the matching cudaFree.
 *   A      device f32 [M][K]          Wq  device int8 [K][N], row-major (QTensor.q layout)
 *   Wscale device f32 [N]             C   device f32 [M][N], written
 *   stream a cudaStream_t (NULL: the default stream); the call only enqueues work.
 * M = 0 or N = 0 enqueue nothing; K = 0 writes zeros (A and Wq may then be NULL).
 * It allocates nothing: its scratch (split-K int32 sums, counters and the row's
 * activation scale) is one fixed __device__ array of 513 KiB inside the library,
 * held by every GPU that loads it until the process exits; hence N <= 131072
 * (larger N is rejected with LLMQ_ERR_ARG, nothing launched).  Every call looks
 * up that array's address (cudaGetSymbolAddress) with the caller's device
 * current; the first call on a device also loads it, so make that first call
 * before any stream capture.  All calls share the array and each clears the
 * words it sums into: calls that overlap on the GPU (other streams, other
 * threads) race and must be serialised by the caller.  Returns 0 or an error
 * code. */
int qmatmul_device_noalloc(const float *A, int M, int K, const signed char *Wq, const float *Wscale, int N,
                           float *C, void *stream);

/* ========================================================================= */
/* Serving operators on device memory (no counterpart in the reference)       */
/* ========================================================================= */
/* What a server of many sequences needs next to the decode step: keys and
 * values in pages, tables of them built on the GPU, the pages' writer,
 * attention of one new token a row over them, and one sampler call for a batch
 * of logits rows.
 *
 * Each call takes descriptors of buffers the caller holds on the current GPU
 * and only enqueues work on `stream` (a cudaStream_t; NULL: the default
 * stream).  Nothing is allocated or kept: a call may be captured into a CUDA
 * graph, and calls on different streams may overlap unless they share an output
 * or a workspace.  Pointers marked "or NULL" are optional.  Sizes, strides and
 * null pointers are checked on the host, and so is that every array starts on
 * one of its elements and is memory of the current GPU; a call that fails one of these checks returns
 * LLMQ_ERR_ARG and enqueues nothing.  n_rows and n_seqs stay below 2^31 - 4096,
 * a row's elements below 2^31.  Values that only the GPU sees (lengths,
 * page ids, slots, positions) are checked there: an entry out of range is left
 * out and its flag is OR'ed into *status (a device int the caller has zeroed, or
 * NULL).  Unused descriptor fields must be zero.  Strides count elements.
 * Returns 0 or an error code. */

/* element types */
enum { LLMQ_F32 = 0, LLMQ_F16 = 1, LLMQ_BF16 = 2 };

/* flags of a status word */
enum {
  LLMQ_PAGED_BAD_LEN = 1,   /* a length below 0 or past the table's row */
  LLMQ_PAGED_NO_PAGES = 2,  /* free pages ran out */
  LLMQ_PAGED_NO_ROWS = 4,   /* more rows than max_rows */
  LLMQ_PAGED_BAD_PAGE = 8,  /* a page id outside the pool, or missing */
  LLMQ_PAGED_BAD_SLOT = 16, /* a slot past the pool */
  LLMQ_PAGED_BAD_POS = 32   /* a position outside the angle tables */
};

/* A pool of pages of keys and values.  Element (page, token, head, d) of k is
 * k[page * page_stride + token * token_stride + head * head_stride + d], the
 * same for v, so [page][token][head][d] and [page][head][token][d] pools are
 * both described.  k and v start on 16 bytes and the strides are multiples of
 * 16 bytes.  Slot s is token s % page_size of page s / page_size. */
typedef struct {
  void *k, *v;
  int dtype;
  int n_pages, page_size; /* n_pages * page_size < 2^31 */
  int n_kv, head_dim;     /* head_dim: a multiple of 8, at most 256 */
  int reserved;
  long long page_stride, token_stride, head_stride;
} LlmqPagedKV;

/* Block tables and slot maps of one step, from the requests' lengths.
 * Request b has cached[b] tokens in its pages (table row b, the first
 * ceil(cached[b] / page_size) entries) and brings added[b] more.  The pages it
 * lacks are taken from free_pages in the order of the requests, starting at
 * free_pages[*free_head], and written into its row.  The step's rows are the
 * added tokens of request 0, then of request 1, and so on.
 *   lens[b]   cached + added                first[b]  first row of request b; first[n_seqs]: rows in all
 *   slots[r]  the row's slot (-1: padding)  positions[r]  its position in the sequence (-1)
 *   seqs[r]   its request (-1)              spans[r]  positions[r] + 1: what the row may attend (0)
 * Rows from first[n_seqs] to max_rows are padding.  *next_head receives the
 * position after the last page taken; it may be free_head itself, and lens may
 * be cached.  A request that cannot be served adds nothing (its lens stay
 * cached): one whose lengths are below 0 or pass the row's max_pages, whose
 * rows (counted over the requests of valid lengths before it) pass max_rows, or
 * whose pages (counted over the requests with rows before it) pass n_free; a
 * request that needs no page is not held up by the last.  A request whose
 * cached length is itself out of range gets lens 0. */
typedef struct {
  int n_seqs, page_size, max_pages, max_rows, n_free;
  int reserved;
  const int *cached, *added;  /* [n_seqs] */
  const int *free_pages;      /* [n_free] */
  const int *free_head;       /* or NULL: 0 */
  int *table;                 /* [n_seqs][table_stride] */
  long long table_stride;
  int *lens, *first;          /* [n_seqs], [n_seqs + 1] */
  long long *slots;           /* [max_rows] */
  int *positions, *seqs, *spans; /* [max_rows], each or NULL */
  int *next_head;             /* or NULL */
  int *status;                /* or NULL */
} LlmqPagedPlan;
int llmq_paged_plan(const LlmqPagedPlan *a, void *stream);

/* Writes a step's keys and values into their slots, and rotates q and k
 * (rope.c:48-68: pairs (d, d + head_dim / 2), in f32) when angle tables are
 * given.  Row r of k and v holds n_kv heads of head_dim, of q n_heads; rows are
 * *_stride apart, so the three may be parts of one packed row.  q_out may be q.
 * Values are rounded once, to the pool's type (q_out: to dtype).  A row whose
 * slot is below 0 is left out (q_out keeps what it held).  Two rows with one
 * slot leave either's values there. */
typedef struct {
  int n_rows, n_heads; /* n_heads: 0 without q */
  int dtype;           /* of q, k, v and q_out */
  int rope_len;        /* positions in the angle tables */
  const void *q, *k, *v;
  long long q_stride, k_stride, v_stride;
  void *q_out;
  long long q_out_stride;
  const long long *slots;  /* [n_rows] */
  const int *positions;    /* [n_rows]; or NULL without tables */
  const float *rope_cos, *rope_sin; /* [rope_len][head_dim / 2], or both NULL */
  int *status;             /* or NULL */
} LlmqPagedAppend;
int llmq_paged_append(const LlmqPagedKV *kv, const LlmqPagedAppend *a, void *stream);

/* Attention of one query row a sequence over a paged cache: row r attends
 * positions [max(0, n - window), n), n = lens[r] (window 0: from 0), of the
 * sequence in table row seqs[r] (NULL: row r):
 *   out = sum_p exp(s_p - m) v_p / sum_p exp(s_p - m),  s_p = scale * <q, k_p>
 * and lse[r][h] = m + log sum_p exp(s_p - m).  n_heads / n_kv query heads share
 * a KV head.  q is in dtype; the pool has the same type, or any type when dtype
 * is LLMQ_F32.  Products are exact, scores, maxima, sums and the output are
 * formed in f32 and rounded once; over a 16-bit pool the weights multiply the
 * values as sums of 16-bit terms (16 bits of a weight for bf16 rows, 22 for f16
 * pools, 24 for f32 rows over bf16).  The result depends on the batch only in
 * the order of its sums.  A row without positions gives zeros and lse -infinity;
 * a head with a NaN or +infinite score (of NaN or infinities in its q or used
 * keys) gives NaN for both.  Positions on a page outside the pool are left out.
 * What the pool holds past a row's length is never read into a result.  out may
 * not overlap q.  scale 0 stands for 1 / sqrt(head_dim).  The workspace need not
 * be initialised; calls that may overlap need one each. */
typedef struct {
  int n_rows, n_heads;
  int dtype;     /* of q and out */
  int window;
  int max_pages; /* entries of a table row; max_pages * page_size < 2^31 - 4096 */
  int n_seqs;    /* table rows */
  float scale;
  int reserved;
  const void *q;          /* [n_rows][n_heads][head_dim], rows q_stride apart */
  long long q_stride;
  void *out;              /* as q; rows out_stride apart */
  long long out_stride;
  float *lse;             /* [n_rows][n_heads], or NULL */
  const int *table;       /* [n_seqs][table_stride] page ids */
  long long table_stride;
  const int *seqs;        /* [n_rows], or NULL */
  const int *lens;        /* [n_rows] */
  void *workspace;        /* 16-byte aligned; llmq_paged_attention_workspace bytes */
  size_t workspace_bytes;
  int *status;            /* or NULL */
} LlmqPagedAttention;
int llmq_paged_attention(const LlmqPagedKV *kv, const LlmqPagedAttention *a, void *stream);
/* Bytes of workspace such a call needs on any sm_100 GPU (0 on bad sizes, with
 * the error set). */
size_t llmq_paged_attention_workspace(int n_rows, int n_heads, int n_kv, int head_dim);

/* Draws one token a row from given random numbers, by the rules of sample_token
 * (sampler.c:60-115) with min-p added.  With w_j = exp((l_j - max l) / T) and
 * the tokens in order of falling logit (the lower index first among equal
 * ones), kept is the shortest of: the first top_k (off: <= 0 or >= vocab); those
 * with w >= min_p (off: <= 0; above 1 counts as 1); and the first tokens whose
 * sum of w reaches top_p of the whole row's (off: outside (0, 1)).  The token
 * drawn is the first one, in that order, at which the sum of w reaches u times
 * the kept sum; u is clamped to [0, 1] (NaN: 0).  A temperature that is not above
 * 0 (NaN too) takes the first largest logit.  Each w is rounded to a multiple of
 * 2^-S, S = min(50, 62 - ceil(log2 vocab)): one below 2^-(S+1) counts as nothing.
 * Sums of those are exact, the same in any order, so a row's token does not depend
 * on the batch it is in; a sum is within vocab * 2^-S of the real one (half of it
 * from rounding, 2^-29 at 128256 tokens; the rest covers the exponential), and
 * only a border nearer than that to a choice may fall to either neighbour.  A NaN
 * or -infinite logit is never drawn; a row of nothing else gives id -1 and logprob
 * -infinity; among +infinite logits the weights are equal.
 * logprobs[r] is the log of the drawn token's share of the kept sum (0 for the
 * greedy choice). */
typedef struct {
  int n_rows, vocab; /* vocab: at most 2^20 */
  int dtype;
  int reserved;
  const void *logits;        /* [n_rows][vocab], rows `stride` apart */
  long long stride;
  const float *temperature;  /* [n_rows], or NULL: 1 */
  const int *top_k;          /* [n_rows], or NULL: off */
  const float *top_p, *min_p; /* [n_rows], each or NULL: off */
  const float *u;            /* [n_rows] random numbers in [0, 1) */
  int *ids;                  /* [n_rows] */
  float *logprobs;           /* [n_rows], or NULL */
} LlmqSampleRows;
int llmq_sample_rows(const LlmqSampleRows *a, void *stream);

/* ---- batches of a model with these operators ---- */

/* Settings of llmq_sample_rows for each sequence, in host memory; a null array is
 * off (temperature: 1).  u is needed. */
typedef struct {
  const float *temperature;
  const int *top_k;
  const float *top_p, *min_p;
  const float *u;
} LlmqSampling;

/* As q_llama_decode_batch_argmax, with each next token drawn by llmq_sample_rows
 * from its row's logits: ids[b] from s->u[b] and the settings of sequence b.
 * Not under tensor parallelism.  Returns 0 or an error code. */
int q_llama_decode_batch_sample(const QLlamaModel *m, LlamaKV **kvs, const int *tokens, int B, const LlmqSampling *s,
                                int *ids);

/* A paged cache of up to max_seqs sequences of a model: n_pages pages of
 * page_size positions (of every layer), shared out as the sequences grow, in
 * place of one max_seq cache a sequence (n_pages * page_size < 2^31 - 4096).
 * dtype is the pages' type; sequences start empty.  head_dim must be a multiple
 * of 8, at most 256.  Not under tensor parallelism.  NULL on error.  The cache
 * belongs to the model: freeing the model frees it (the handle is then invalid). */
typedef struct LlmqPagedCache LlmqPagedCache;
LlmqPagedCache *q_llama_paged_create(const QLlamaModel *m, int n_pages, int page_size, int max_seqs, int dtype);
void q_llama_paged_free(LlmqPagedCache *c);
/* Positions sequence seq holds, or -1 on error; pages that no sequence holds. */
int q_llama_paged_len(const LlmqPagedCache *c, int seq);
int q_llama_paged_free_pages(const LlmqPagedCache *c);
/* Empties sequence seq: its pages are free again.  Returns 0 or an error code. */
int q_llama_paged_reset(LlmqPagedCache *c, int seq);

/* One step of a batch: sequence b takes added[b] tokens (0: it sits out; 1: a
 * decode step; more: a prompt or a piece of one), listed in `tokens` sequence
 * after sequence.  All rows go through the layers together: llmq_paged_plan,
 * then in each layer llmq_paged_append and llmq_paged_attention, and one
 * llmq_sample_rows (s null: the greedy choice) for the last row of every sequence
 * that took any.  ids[b] receives sequence b's next token (-1 if it sat out);
 * `logits`, if given, the rows ids came from, one below the other for the
 * sequences that took tokens, in their order.  Attention runs as documented at
 * llmq_paged_attention: unlike q_llama_decode_batch it does not keep the
 * reference's order of additions, so logits are near that path's, not equal bit
 * for bit.  Each row of a prompt reads its sequence's keys and values on its own,
 * so a prompt's reads grow with the square of its length.  An error leaves the
 * sequences as they were (LLMQ_ERR_OOM: pages, or memory for so many rows, ran
 * out); after one of the GPU in the middle of a step the cache answers
 * LLMQ_ERR_STATE until it is freed.  Returns 0 or an error code. */
int q_llama_paged_step(const QLlamaModel *m, LlmqPagedCache *c, const int *added, const int *tokens,
                       const LlmqSampling *s, int *ids, Tensor *logits);

#ifdef __cplusplus
}
#endif

#endif /* LLMQ_CUDA_H */
