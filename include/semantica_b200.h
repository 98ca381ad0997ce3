/*
 * semantica_b200.h — C ABI of libsemantica_b200.so, the B200 (sm_100a)
 * implementation of go-semantica's two data-parallel hot paths:
 *
 *   1. the EmbeddingGemma INT8 forward pass behind rt.Embed
 *      (internal/runtime.(*Model).ForwardWithDim, model.go:661-666), and
 *   2. search/brute's quantised scan + top-k behind Index.SearchVector and
 *      the BRUT v1 Serializer (search/brute/index.go, storage.go).
 *
 * Plain C types only: pointers, sizes, status codes. Every call returns a
 * SEM_* status; on failure sem_last_error() returns a message that matches the
 * reference's error string where the reference has one. No call keeps a
 * pointer to caller memory after it returns (the cgo rule): inputs are copied.
 * A context is bound to one GPU; calls on one context are serialised.
 *
 * Citations are "file:line" inside the go-semantica source tree.
 */
#ifndef SEMANTICA_B200_H
#define SEMANTICA_B200_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* ---- status codes ---- */
#define SEM_OK 0
#define SEM_EINVAL 1    /* invalid argument (reference-style message in sem_last_error) */
#define SEM_EDEVICE 2   /* CUDA error */
#define SEM_ENOMEM 3    /* device or host allocation failed */
#define SEM_EFORMAT 4   /* malformed GGUF or BRUT bytes */
#define SEM_ENOTFOUND 5 /* tensor / id not found */
#define SEM_EINTERNAL 6 /* a host-side failure inside the library (e.g. a thread could not start) */

typedef struct sem_context sem_context;
typedef struct sem_model sem_model;
typedef struct sem_index sem_index;
typedef struct sem_q8_weight sem_q8_weight;
typedef struct sem_group sem_group;
typedef struct sem_adapter_plan sem_adapter_plan;
typedef struct sem_lowrank sem_lowrank;
typedef struct sem_block_norm sem_block_norm;
typedef struct sem_model_adapters sem_model_adapters;

/* Message of the last failed call on this thread (never NULL). A Go caller
 * holds its OS thread (runtime.LockOSThread) from the failing call until it
 * has read the message: a goroutine may change threads between cgo calls. */
const char *sem_last_error(void);

/* Number of visible CUDA devices. */
int sem_device_count(int *out);

/* A context owns one device, one stream and the device workspaces. */
int sem_context_create(int device, sem_context **out);
int sem_context_destroy(sem_context *ctx);
/* The context's CUDA stream, as a cudaStream_t. */
void *sem_context_stream(sem_context *ctx);

/* ------------------------------------------------------------------------
 * Model: replaces internal/runtime.LoadModel / loadModel (model.go:233-315)
 * ---------------------------------------------------------------------- */

/* Mirrors internal/runtime.ModelConfig (model.go:16-31). */
typedef struct sem_model_config {
  int32_t vocab_size, embed_dim, num_layers, num_heads, num_kv_heads, head_dim, interm_dim, max_seq_len;
  float norm_eps, rope_base, attention_scale;
} sem_model_config;

/* A GGUF tensor as internal/gguf.Reader exposes it (reader.go:23-30,
 * :332-346): dims are GGUF ne[] (ne0 contiguous), dtype is the GGUF type id
 * (0 F32, 8 Q8_0), data points at the tensor bytes (e.g. into the mmap). */
typedef struct sem_tensor_view {
  const char *name;
  uint32_t dtype;
  uint32_t n_dims;
  uint64_t dims[4];
  const void *data;
  uint64_t nbytes;
} sem_tensor_view;

/* Uploads the model named by `tensors` (token_embd.weight, output_norm.weight,
 * blk.N.{attn_norm,attn_q,attn_k,attn_v,attn_output,attn_q_norm,attn_k_norm,
 * post_attention_norm,ffn_norm,ffn_gate,ffn_up,ffn_down,post_ffw_norm}.weight,
 * model_int8.go:54-119) to the context's device, repacking every Q8_0 tensor
 * into an int8 plane and an fp32 block-scale plane. The caller's bytes may be
 * released when the call returns. Replaces loadWeights + loadLayerINT8
 * (model.go:520-552, model_int8.go:54-119). */
int sem_model_load(sem_context *ctx, const sem_model_config *cfg, const sem_tensor_view *tensors, int32_t n_tensors,
                   sem_model **out);

/* Convenience: parses a GGUF v3 file the way internal/gguf + parseConfig do
 * (reader.go:98-178, model.go:424-517) and calls sem_model_load. */
int sem_model_load_gguf(sem_context *ctx, const char *path, sem_model **out);

int sem_model_config_get(const sem_model *model, sem_model_config *out);
int sem_model_free(sem_model *model);

/* ------------------------------------------------------------------------
 * Embedding forward: replaces (*Model).ForwardWithDim (model.go:661-666 →
 * model_int8.go:148-256), batched. The reference runs one sequence per call
 * and fans calls out over goroutines (pkg/ggufembed/api.go:237-295); here one
 * call carries every sequence of a request.
 * ---------------------------------------------------------------------- */

/* ids: packed token ids of n_seqs sequences; offsets: n_seqs+1 prefix offsets
 * into ids; dims: per-sequence output dimension (1..embed_dim; NULL = embed_dim
 * for all); out: packed outputs, sequence s at sum(dims[0..s-1]), each the
 * mean-pooled, L2-normalised first dims[s] channels.
 * Errors (reference strings): "empty input", "sequence too long: %d > %d",
 * "token ID out of range: %d", "target dimension %d out of range (1..%d)". */
int sem_embed(sem_model *model, const int32_t *ids, const int32_t *offsets, int32_t n_seqs, const int32_t *dims,
              float *out);

/* Device-resident variant (no host copies): d_ids on the device, h_offsets on
 * the host, d_out on the device (n_seqs x dim). Enqueued on `stream` (NULL =
 * the context stream); returns without synchronising, so errors the device
 * detects (a token id outside the vocabulary, a timed-out pipeline wait)
 * surface through sem_model_check. */
int sem_embed_device(sem_model *model, const int32_t *d_ids, const int32_t *h_offsets, int32_t n_seqs, int32_t dim,
                     float *d_out, void *stream);

/* The request pipeline (no reference counterpart; it stands in for the
 * reference's one goroutine per prompt, pkg/ggufembed/api.go:237-295, at the
 * level of whole requests). sem_embed_submit checks a request exactly as
 * sem_embed does, copies its ids and metadata into one of the model's two
 * request slots (pinned host staging), enqueues the upload, the forward and
 * the download of its outputs, and returns a ticket without waiting.
 * sem_embed_wait(ticket) blocks until that request is done and writes its
 * outputs (sem_embed's layout) to `out`. While one request runs on the
 * device the host prepares (tokenises, submits) the next. At most two
 * requests are in flight: a third submit fails with SEM_EINVAL until one is
 * waited for. Requests run in submission order; each ticket is waited for
 * once. Errors the device reports (a timed-out pipeline wait) are returned by
 * sem_embed_wait. */
int sem_embed_submit(sem_model *model, const int32_t *ids, const int32_t *offsets, int32_t n_seqs,
                     const int32_t *dims, uint64_t *ticket);
int sem_embed_wait(sem_model *model, uint64_t ticket, float *out);

/* Waits for the model's device to finish every forward enqueued so far and
 * reports what the device recorded since the last check (or sem_embed call):
 * SEM_EINVAL "token ID out of range: ..." for a device-resident id outside the
 * vocabulary (its embedding row was written as zeros), SEM_EDEVICE when a
 * tensor-core pipeline wait timed out (that kernel returned early and its
 * output is incomplete). Clears the record. No reference counterpart: the
 * reference validates ids on the host (model_int8.go:167-178). */
int sem_model_check(sem_model *model);

/* Model-faithful mode. The reference runs full bidirectional attention in
 * every layer and has no dense head (model_int8.go:235-255, :500); the
 * EmbeddingGemma architecture has both, and this mode restores them. It has
 * no counterpart in the reference and is off by default (sem_embed computes
 * the reference's forward).
 *   sliding_window: in sliding layers query i sees keys j with
 *     |i - j| <= sliding_window / 2 (0: every layer sees every key);
 *   swa_pattern: layer l (0-based) is a global layer when (l + 1) % swa_pattern
 *     == 0, a sliding layer otherwise (EmbeddingGemma: window 512, pattern 6);
 *   rope_base_swa: RoPE base of the sliding layers (0: the model's rope_base);
 *   dense_head: after output_norm and mean pooling of every channel, the
 *     dense_2.weight (embed -> mid) and dense_3.weight (mid -> embed) Q8_0
 *     projections, each input quantised per sequence like every projection of
 *     the forward; then the first dims[s] outputs, L2-normalised. The weights
 *     are read at load when the tensors are present. */
typedef struct sem_faithful_config {
  int32_t sliding_window, swa_pattern;
  float rope_base_swa;
  int32_t dense_head;
} sem_faithful_config;
/* cfg NULL (or all zero): the reference's forward. Errors: SEM_EINVAL for
 * negative fields or a dense head the model has no weights for. */
int sem_model_set_faithful(sem_model *model, const sem_faithful_config *cfg);

/* ------------------------------------------------------------------------
 * Several GPUs of one host as one embedding engine. The reference fans the
 * sequences of a request out over goroutines (pkg/ggufembed/api.go:237-295);
 * a group fans them out over devices: one context and one model replica per
 * device, each request split by token count (longest sequence first to the
 * device holding the fewest tokens) and embedded on every device at once from
 * one host thread per device. No collective: replicas share nothing.
 * ---------------------------------------------------------------------- */

/* Loads the model on each of the n_devices distinct devices (in parallel). */
int sem_group_load(const int32_t *devices, int32_t n_devices, const sem_model_config *cfg,
                   const sem_tensor_view *tensors, int32_t n_tensors, sem_group **out);
int sem_group_load_gguf(const int32_t *devices, int32_t n_devices, const char *path, sem_group **out);
int sem_group_size(const sem_group *group, int32_t *out);
int sem_group_config_get(const sem_group *group, sem_model_config *out);
/* sem_model_set_faithful on every replica, or on none: when one replica fails,
 * those already switched return to their previous setting and the error names
 * the device. */
int sem_group_set_faithful(sem_group *group, const sem_faithful_config *cfg);
/* sem_embed's contract (same arguments, errors and output layout); the
 * request is validated on the host before any device starts, and a device's
 * error is returned as "device N: <message>". One request at a time per
 * group; concurrent callers wait. */
int sem_group_embed(sem_group *group, const int32_t *ids, const int32_t *offsets, int32_t n_seqs,
                    const int32_t *dims, float *out);
int sem_group_free(sem_group *group);

/* Per-stage device timing of the forward pass (diagnostics; no reference
 * counterpart). enable != 0 brackets every kernel launch of later forwards
 * with CUDA events on the launching stream. profile_read synchronises the
 * context stream, returns up to `cap` stages (static names, total ms, launch
 * counts) accumulated since the last read, and resets the totals. */
int sem_model_profile(sem_model *model, int32_t enable);
int sem_model_profile_read(sem_model *model, const char **names, float *total_ms, int32_t *launches, int32_t cap,
                           int32_t *n_out);

/* ------------------------------------------------------------------------
 * Isolated Q8_0 x INT8 projection: QuantizeSymmetricINT8Into + MatMulQ8_0INT8
 * (internal/kernels/quantize.go:29-69, :346-458).
 * ---------------------------------------------------------------------- */

/* w_q8: raw Q8_0 bytes of an [n_out rows x k_in] weight (GGUF dims {k_in, n_out}). */
int sem_q8_weight_create(sem_context *ctx, const void *w_q8, int32_t k_in, int32_t n_out, sem_q8_weight **out);
int sem_q8_weight_free(sem_q8_weight *w);
/* Device pointers: d_a fp32 [m x k_in] -> d_c fp32 [m x n_out], one activation
 * scale for the whole of d_a as in the reference; d_codes and d_absmax (one
 * uint32) are caller-provided scratch. d_codes holds the m x k_in INT8 codes
 * as fp16 (the tensor cores' operand type; 2 * m * k_in bytes, 16-byte
 * aligned). Enqueued on `stream`. */
int sem_q8_gemm(sem_q8_weight *w, const float *d_a, int32_t m, float *d_c, void *d_codes, uint32_t *d_absmax,
                void *stream);

/* MatMulQ8_0INT8 alone (quantize.go:346-458) on activations already quantised
 * by QuantizeSymmetricINT8Into: d_codes holds the m x k_in INT8 codes as fp16
 * (16-byte aligned), *d_absmax the float32 bit pattern of the absmax they were
 * quantised with (scale = absmax / 127, as quantize.go:60-61); d_c fp32
 * [m x n_out]. Enqueued on `stream`. */
int sem_q8_matmul_int8(sem_q8_weight *w, const void *d_codes, const uint32_t *d_absmax, int32_t m, float *d_c,
                       void *stream);

/* Which kernel the Q8_0 projections use (process-wide, every model and
 * weight). Three kernels exist:
 *   - the CUDA-core kernel computes the reference's VNNI inner loop exactly
 *     (simd_amd64.s:241-304: 8 float32 lane accumulators, each a fused
 *     multiply-add of an exact 4-product int32 partial and the block scale,
 *     then the reference's horizontal sum and the unfused inputScale
 *     multiply): bit-identical to the reference's default amd64 build;
 *   - the per-block tensor-core kernel sums each 32-element block exactly and
 *     scales it in float32, accumulating the blocks in another order;
 *   - the split-plane tensor-core kernel folds the block scales into two fp16
 *     weight planes (one TMEM drain per tile, the fastest at scale) and differs
 *     from the reference's sums in the last float32 bits.
 * sem_embed packs sequences of >= 128 tokens first. Shorter sequences (while
 * a batch holds at most 4096 of their tokens; beyond that they take the
 * tensor-core kernels as long rows do) take the CUDA-core kernel (and a
 * float32 attention in the reference's order), so their embeddings are
 * bit-identical to the reference's; long-sequence rows
 * take a tensor-core kernel (mean pooling over many tokens keeps the
 * difference within the reference's own spread between its builds).
 *   SEM_Q8_PATH_AUTO (default): long-sequence rows take the split-plane kernel
 *     when its 128 x 256-token tiles fill at least half the SMs, else the
 *     per-block kernel; sem_q8_gemm / sem_q8_matmul_int8 take the CUDA-core
 *     kernel below 128 rows, then the same rule;
 *   SEM_Q8_PATH_BLOCK: the per-block kernel everywhere;
 *   SEM_Q8_PATH_SPLIT: the split-plane kernel for long-sequence rows (all
 *     rows for sem_q8_gemm) whatever their count;
 *   SEM_Q8_PATH_SPLIT_ALL: the split-plane kernel for every row (testing);
 *   SEM_Q8_PATH_EXACT: the CUDA-core kernel for every row (bit-exact
 *     projections at any length, slower than the tensor cores at scale).
 * A tuning and testing switch with no counterpart in the reference. Returns
 * the previous setting, or -1 for an unknown mode. */
#define SEM_Q8_PATH_AUTO 0
#define SEM_Q8_PATH_BLOCK 1
#define SEM_Q8_PATH_SPLIT 2
#define SEM_Q8_PATH_SPLIT_ALL 3
#define SEM_Q8_PATH_EXACT 4
int sem_q8_path(int32_t mode);

/* sem_q8_gemm without caller scratch, for callers that cannot allocate device
 * memory (a host runtime that owns the whole device pool and passes only input
 * and output buffers, or a request path with a memory budget fixed at start-up
 * where an allocation may neither grow nor fail). It has no counterpart in the
 * reference. The codes and the absmax word live in a static device array of
 * 16 MiB + 256 bytes that every GPU loading the library holds until exit, so
 * m * k_in must not exceed 8 Mi (8,388,608) elements (larger calls fail with
 * SEM_EINVAL); m == 0 is a no-op, as for sem_q8_gemm. The kernel choice is
 * sem_q8_gemm's (sem_q8_path). The call performs no allocation. The first
 * call on a device resolves the array's address on that device
 * (cudaGetSymbolAddress), which loads the library's device code there and may
 * synchronise the device; the array's 16 MiB are committed then, not when the
 * library is loaded. Make that first call (a warm-up call will do) at start-up,
 * before the host runtime reserves its device pool and before any stream
 * capture. All calls share the one array: calls that overlap on the GPU (other
 * streams, other threads) race on it. Enqueued on `stream` (NULL = the
 * weight's context stream). */
int sem_q8_gemm_noalloc(sem_q8_weight *w, const float *d_a, int32_t m, float *d_c, void *stream);

/* ------------------------------------------------------------------------
 * Adapters of many requests beside one shared base model. No counterpart in
 * the reference, which serves one model without adapters. A batch is packed
 * sequences, as for sem_embed; each sequence names an adapter or none. The
 * plan says which adapter every row uses; the operators below go by it. A
 * plan, a bank and a block norm belong to one device; the calls take device
 * pointers, are enqueued on `stream` (NULL = the handle's context stream) and
 * return without synchronising. They allocate nothing and keep no state, so
 * calls may overlap, on one stream or several, and may be captured into CUDA
 * graphs. On the context's own stream they take their turn with the context's
 * other calls (sem_embed keeps it until its outputs are there).
 * ---------------------------------------------------------------------- */

/* Element types of the operators' rows and weights. */
#define SEM_DTYPE_F32 0
#define SEM_DTYPE_F16 1
#define SEM_DTYPE_BF16 2

/* A plan for batches of up to max_rows rows in up to max_seqs sequences. */
int sem_adapter_plan_create(sem_context *ctx, int64_t max_rows, int32_t max_seqs, sem_adapter_plan **out);
/* Sets the batch (host arrays, copied): sequence s is rows
 * [offsets[s], offsets[s+1]) (offsets[0] = 0, empty sequences allowed) and
 * uses adapters[s], -1 for none; several sequences may use one adapter. The
 * tables are uploaded on `stream`: work that uses the plan is ordered after
 * the call there, and work enqueued earlier that still reads the plan's
 * previous batch must be on the same stream or done. Not inside a stream
 * capture; a captured operator reads the batch that the plan holds when the
 * graph is replayed (a plan set to another batch needs no new capture; the
 * caller keeps its buffers as large as that batch needs, and its adapter
 * indexes within the bank: a row of an adapter that the bank does not have is
 * then treated as a row without one). */
int sem_adapter_plan_set(sem_adapter_plan *plan, const int32_t *offsets, const int32_t *adapters, int32_t n_seqs,
                         void *stream);
int sem_adapter_plan_free(sem_adapter_plan *plan);

/* Low-rank adapters of one projection (k_in -> n_out, each 1..65536): adapter
 * i has weights a[i] [ranks[i]][k_in] and b[i] [n_out][ranks[i]] (host
 * pointers, row-major, of element type dtype, copied) and the factor
 * scales[i]; ranks 0..128, 0 for an adapter that leaves this projection as it
 * is (its pointers are not read). A bank keeps its weights as given and as
 * tiles for every type of x: an fp16 adapter of rank 16 of 768 x 768 takes 270
 * KB of device memory, 5.5 times its weights (ranks are padded to 32 in b's
 * tiles: of rank 8 184 KB, 7.5 times). */
int sem_lowrank_create(sem_context *ctx, int32_t k_in, int32_t n_out, int32_t n_adapters, const int32_t *ranks,
                       const float *scales, const void *const *a, const void *const *b, int32_t dtype,
                       sem_lowrank **out);
int sem_lowrank_free(sem_lowrank *w);
/* For every row of the plan's batch, with its sequence's adapter i:
 *   y = base + scales[i] * (x a[i]^T) b[i]^T,
 * and y = base for rows without an adapter. x: k_in values a row; base and y:
 * n_out values a row of y's type, base is normally the shared projection's
 * output (sem_q8_gemm). base may be y itself, or NULL for zeros; apart from
 * that y overlaps neither x nor base. Row strides ldx, ld_base, ldy in
 * elements, 0 for packed rows; any stride and any element-aligned address is
 * allowed (rows that start on 16 bytes load fastest). Types: x F32 with y
 * F32; x F16 or BF16 with y of the same type or F32. Products and sums are
 * held in float32, with x, the weights and the rank-wide intermediate carried
 * to at least 21 bits; the result is rounded once, to y's type. Infinities and
 * NaN in x give what the formula gives and stay in their rows (the weights are
 * finite). The same call gives the same bits again, and with one kernel for
 * both (sem_lowrank_path) a row's bits do not depend on the batch around it;
 * SEM_LOWRANK_PATH_AUTO goes by the whole call's work, so there they may, within
 * the above. */
int sem_lowrank_apply(sem_lowrank *w, sem_adapter_plan *plan, const void *d_x, int32_t x_dtype, int64_t ldx,
                      const void *d_base, int64_t ld_base, void *d_y, int32_t y_dtype, int64_t ldy, void *stream);
/* The same beside sem_q8_matmul_int8: x = code * (absmax / 127), d_codes the
 * rows x k_in INT8 codes as fp16, d_absmax the float32 bit patterns of the
 * absmax they were quantised with. n_absmax says how many and what they
 * belong to: 1, one for every row; n_seqs, one per sequence of the plan; or
 * by name, SEM_ABSMAX_ALL_ROWS and SEM_ABSMAX_PER_SEQUENCE, whatever the
 * plan's batch. A captured call keeps the meaning that it was captured with.
 * Where a capture meets a plan of one sequence, n_absmax = 1 could be either,
 * and is refused: name it (a replay may find another batch, for which
 * d_absmax then has to hold a scale per sequence, or one). */
#define SEM_ABSMAX_ALL_ROWS (-2)
#define SEM_ABSMAX_PER_SEQUENCE (-3)
int sem_lowrank_apply_int8(sem_lowrank *w, sem_adapter_plan *plan, const void *d_codes, const uint32_t *d_absmax,
                           int32_t n_absmax, const float *d_base, int64_t ld_base, float *d_y, int64_t ldy,
                           void *stream);
/* Which kernel runs the low-rank products (process-wide):
 *   SEM_LOWRANK_PATH_AUTO (default): the tensor cores, or the CUDA cores where
 *     the whole call is too little work to fill the tensor cores' pipeline;
 *   SEM_LOWRANK_PATH_CUDA_CORES, SEM_LOWRANK_PATH_TENSOR: always these.
 * A tuning and testing switch, like sem_q8_path. Returns the previous setting,
 * or -1 for an unknown mode. */
#define SEM_LOWRANK_PATH_AUTO 0
#define SEM_LOWRANK_PATH_CUDA_CORES 1
#define SEM_LOWRANK_PATH_TENSOR 2
int sem_lowrank_path(int32_t mode);
/* Waits for the device and reports what its calls recorded since the last
 * check: SEM_EDEVICE when a tensor-core pipeline wait timed out (that call's
 * output is incomplete). */
int sem_lowrank_check(sem_lowrank *w);

/* The norms after a block and before the next one, fused with the block's
 * gate and residual scale (host pointers, copied): post_w, pre_w [dim] (NULL:
 * that norm is left out), gates [n_adapters][dim] (NULL: 1), scales
 * [n_adapters] (NULL: 1), dim 1..16384. */
int sem_block_norm_create(sem_context *ctx, int32_t dim, float eps, const float *post_w, const float *pre_w,
                          int32_t n_adapters, const float *gates, const float *scales, sem_block_norm **out);
int sem_block_norm_free(sem_block_norm *b);
/* For every row, with its adapter i (plan NULL: i = 0 for every row; rows
 * without an adapter: gate and scale 1):
 *   h_out = scales[i] * h + gates[i] * (rmsnorm(o) * post_w)
 *   y     = rmsnorm(h_out) * pre_w        (from h_out before its rounding)
 * rmsnorm(v) = v / sqrt(mean(v^2) + eps), in float32; o itself without
 * post_w, no y (d_y is not used) without pre_w. o and y are of type dtype, h
 * and h_out of type h_dtype (dtype, or F32). h_out may be h, y may be o; no
 * other overlap. `rows` is the plan's row count when there is a plan; a
 * captured call keeps it, so its plan may be set to batches of that many rows.
 * Strides as for sem_lowrank_apply. */
int sem_block_norm_run(sem_block_norm *b, sem_adapter_plan *plan, int64_t rows, const void *d_o, int64_t ldo,
                       int32_t dtype, const void *d_h, int64_t ldh, int32_t h_dtype, void *d_h_out, int64_t ld_h_out,
                       void *d_y, int64_t ldy, void *stream);

/* One adapter of a model: tensors named as in a GGUF adapter file,
 *   blk.N.P.weight.lora_a {k_in, rank} and blk.N.P.weight.lora_b {rank, n_out}
 * with P one of attn_q, attn_k, attn_v, attn_output, ffn_gate, ffn_up,
 * ffn_down (type 0 F32, 1 F16 or 30 BF16; any subset of layers and
 * projections, ranks 1..128), and, type F32, the gates and residual scales of
 * a layer's two blocks,
 *   blk.N.attn_residual.gate {embed_dim}, blk.N.attn_residual.scale {1},
 *   blk.N.ffn_residual.gate {embed_dim}, blk.N.ffn_residual.scale {1}.
 * The low-rank products are multiplied by alpha / rank (alpha 0: by 1). */
typedef struct sem_adapter_view {
  const sem_tensor_view *tensors;
  int32_t n_tensors;
  float alpha;
} sem_adapter_view;

/* Uploads n_adapters adapters of `model` (the caller's bytes may be released
 * when the call returns); freed before the model. Errors: SEM_EFORMAT for a
 * tensor with another name, shape or type, or a lora_a without its lora_b. */
int sem_model_adapters_create(sem_model *model, const sem_adapter_view *adapters, int32_t n_adapters,
                              sem_model_adapters **out);
int sem_model_adapters_free(sem_model_adapters *adapters);

/* sem_embed with an adapter for each sequence: use[s] an index, or -1 for the
 * model as it is. One batch carries the sequences of many adapters; the base
 * projections are shared. Every low-rank product reads the INT8 codes that the
 * projection beside it reads, adds to its output before norm, attention or
 * GELU, and a block's gate and residual scale apply where its post norm is
 * added to the residual stream. Otherwise sem_embed's contract. A sequence
 * with use[s] = -1 is embedded by the model as it is (where an adapter has a
 * gate or residual scale, that layer's norm sums are float32 in another order
 * for the whole batch); a batch of none but such runs sem_embed's forward. The
 * low-rank products' float32 rounding may go by the batch's size (see
 * sem_lowrank_apply). Not captured into the model's cached CUDA graphs.
 * Further error: "adapter %d out of range (-1..%d)". */
int sem_embed_adapted(sem_model *model, sem_model_adapters *adapters, const int32_t *ids, const int32_t *offsets,
                      int32_t n_seqs, const int32_t *use, const int32_t *dims, float *out);

/* ------------------------------------------------------------------------
 * Brute-force index: replaces search/brute (builder.go, index.go, storage.go).
 * quant: 0 float32, 1 int8, 2 int16 (brute.QuantizationMode, quant.go:8-15).
 * ---------------------------------------------------------------------- */

/* Builder.AddVector + Build (builder.go:52-127): vectors are normalised
 * (builder.go:129-141) and quantised (quant.go:17-41) on the device.
 * ids must be unique ("brute: duplicate id %d"). */
int sem_index_build(sem_context *ctx, int32_t dim, int32_t quant, const float *vectors, const int32_t *ids,
                    int64_t count, sem_index **out);

/* An index from already-stored rows (codes as Build or Deserialize produce
 * them): data is count x dim of int8 / int16 / float32, in host or device
 * memory. int8 indexes with dim >= 128 search on the tensor cores. */
int sem_index_create(sem_context *ctx, int32_t dim, int32_t quant, const void *data, const int32_t *ids, int64_t count,
                     sem_index **out);

int sem_index_free(sem_index *idx);
int sem_index_count(const sem_index *idx, int64_t *out);
int sem_index_dimension(const sem_index *idx, int32_t *out);
int sem_index_quantization(const sem_index *idx, int32_t *out);

#define SEM_SEARCH_REFERENCE 0 /* fp32 query x (code/127): the reference's own arithmetic */
#define SEM_SEARCH_EXACT 1     /* query quantised like the rows, exact int32 dot products */

/* Index.SearchVector (index.go:29-42) for nq queries (nq x dim floats, not
 * yet normalised; normalize != 0 normalises them first as SearchVector does,
 * 0 treats them as normalised like SearchNormalized, :44-53). Results per
 * query: min(k, count) entries, best first; ties break toward the lower row.
 * out_ids/out_dist are nq x k (unused tail entries: id -1). out_scores (exact
 * mode, may be NULL) receives the int32 scores. Errors: "brute: topK must be
 * positive", "brute: query dimension mismatch: got %d want %d". */
int sem_index_search(sem_index *idx, const float *queries, int32_t nq, int32_t dim, int32_t k, int32_t mode,
                     int32_t normalize, int32_t *out_ids, float *out_dist, int32_t *out_scores);

/* Device-level search of one shard for multi-GPU merges: d_qcodes (exact
 * mode, nq x dim codes of the index's element type) or d_queries (reference
 * mode, normalised floats); writes nq x k 64-bit candidate keys
 * ((order-preserving score << 32) | ~global_row) to d_keys, where global_row =
 * row_base + local row. Enqueued on `stream`. */
int sem_index_search_keys(sem_index *idx, const void *d_queries, int32_t nq, int32_t k, int32_t mode,
                          int64_t row_base, uint64_t *d_keys, void *stream);

/* Merges `lists` candidate-key lists of k per query (d_keys: lists x nq x k)
 * into the best k_out per query. quant selects the distance scale (1: /127^2,
 * 2: /32767^2) for exact-mode keys. Any output may be NULL. */
int sem_topk_merge(sem_context *ctx, const uint64_t *d_keys, int32_t lists, int32_t nq, int32_t k, int32_t k_out,
                   int32_t mode, int32_t quant, int32_t *d_rows, int32_t *d_scores, float *d_dist, void *stream);

/* Quantises normalised queries exactly like stored rows (quant.go:17-41). */
int sem_quantize_queries(const float *queries, int32_t nq, int32_t dim, int32_t quant, void *out_codes);

/* Index.Vector (index.go:162-180): dequantised copy of the row with this id. */
int sem_index_vector(sem_index *idx, int32_t id, float *out);

/* BRUT v1 (storage.go:17-153): 20-byte header {"BRUT", u16 version 1, u16 dim,
 * u32 count, u8 quantization, 7 pad}, int32 ids[count], row-major data; little
 * endian. serialize: pass buf = NULL to get the size in *written. */
int sem_index_serialize(sem_index *idx, void *buf, size_t cap, size_t *written);
int sem_index_deserialize(sem_context *ctx, const void *bytes, size_t n, sem_index **out);

#ifdef __cplusplus
}
#endif
#endif
