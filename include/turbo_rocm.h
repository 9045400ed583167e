/* SPDX-License-Identifier: Apache-2.0
 *
 * The rocm backend's C ABI: libturbo_rocm.so.
 *
 * The drop-in boundary is one symbol, the backend's function table, which
 * the TurboEmbed core lists beside its other backends. Everything else here
 * is the host-side checking the core does before it calls a backend (so a
 * harness without the Rust core checks rows as the core does), operators on
 * device memory for programs that run layers of their own over a session's
 * states, and hooks for tests and measurement, which the core never calls.
 */
#ifndef TURBO_ROCM_H
#define TURBO_ROCM_H

#include "turbo/turbo_seam.h"

#ifdef __cplusplus
extern "C" {
#endif

/* The backend's table, name "rocm". Replaces, for AMD gfx950 GPUs, the
 * reference's turbo_cuda_backend (core/cuda/backend.cpp:3776-3809), and is
 * linked into the core's LINKED list the same way
 * (core/src/backend/mod.rs:338-360, extern static as core/src/cuda.rs:8-17).
 * Every function follows include/turbo/turbo_backend.h:455-627. */
extern const turbo_backend turbo_rocm_backend;

/* The numeric class of BF16 operands with F32 sums: this backend's BF16 tier.
 * The reference defines classes 1, 2, 4 and 8 (turbo_backend.h:226-229); this
 * is the next free bit, which the core's NUMERICS_ALLOWED table
 * (core/src/tuning.rs:32-41) needs for a BF16-stored model. */
#define TURBO_ROCM_NUMERIC_BF16_F32ACC 16u

/* The numeric class of int8 operands with int32 sums, dequantized in F32: a
 * symmetric scale per weight row (output channel) and per token, this
 * backend's I8 tier. It runs for a model whose turbo_backend_model.compute_dtype
 * is TURBO_DTYPE_I8, at MODEL and FASTEST; the reference's only I8 encoder is
 * a compiled Hailo graph (core/hailo/backend.cpp:441-443, 510). */
#define TURBO_ROCM_NUMERIC_I8_I32ACC 32u

/* ---- The core's checks of a write (core/src/session/tokens.rs:274-384) ----
 *
 * turbo_rocm_check_tokens: the rows' shape within max_batch x max_seq, each id
 * under vocab, each type under types (types may be NULL), each mask entry 0
 * or 1 with a 1 in every row, and, when max_tokens is not 0, each row's
 * length through its last live token at most max_tokens. row_stride 0 is seq.
 * Returns TURBO_OK or the status the core returns, with its message. */
int32_t turbo_rocm_check_tokens(uint32_t batch, uint32_t seq, uint32_t row_stride, const int32_t *ids,
                                const int32_t *mask, const int32_t *types, uint32_t max_batch, uint32_t max_seq,
                                uint32_t vocab, uint32_t token_types, uint32_t max_tokens, turbo_error *err);

/* turbo_rocm_check_ranges: count ranges of the rows above (the core's
 * check_ranges, core/src/session/tokens.rs:274-306, for a backend that does
 * not compute mask-0 columns): count 1 to max_ranges, each row under batch,
 * start under end, end at most seq, and a live token inside. */
int32_t turbo_rocm_check_ranges(uint32_t batch, uint32_t seq, uint32_t row_stride, const int32_t *mask,
                                const turbo_token_range *ranges, uint32_t count, uint32_t max_ranges,
                                turbo_error *err);

/* ---- The rerank caller (core/src/tokenizer/pair.rs:27-99,
 * core/src/session/rerank.rs:47-219) ----
 *
 * turbo_rocm_pair_windows: a query and a passage, as token ids, into the
 * encoder windows of the pair template [start] query [end] passage [end]
 * (RoBERTa, roberta != 0: [start] query [end] [end] passage [end], one
 * segment): the query cut to query_tokens on the right, the passage covered
 * by windows of max_tokens - specials - query tokens, stride apart (0:
 * disjoint). Each window is a row of max_tokens ids and types (BERT: type 1
 * from the passage on) padded with id 0, and its length. Writes up to
 * capacity windows and *windows = their number; TURBO_E_CAPACITY when more
 * are needed. Errors as the reference's: field 2 max_tokens, 1 query_tokens,
 * 3 stride. */
int32_t turbo_rocm_pair_windows(const int32_t *query, uint32_t query_len, const int32_t *passage, uint32_t passage_len,
                                int32_t start_id, int32_t end_id, uint32_t roberta, uint32_t query_tokens,
                                uint32_t max_tokens, uint32_t stride, int32_t *ids, int32_t *types, uint32_t *lengths,
                                uint32_t capacity, uint32_t *windows, turbo_error *err);

/* turbo_rocm_rerank_scores: the sequence classification head over n CLS
 * states [n, hidden] F32 (core/src/session/rerank.rs:166-191): the pooler
 * (dense [hidden, hidden] + bias, tanh; skipped when pooler_weight is NULL)
 * and the one-logit classifier, each summed in F64 from its bias and rounded
 * to F32. A non-finite state or logit is TURBO_E_INTERNAL. */
int32_t turbo_rocm_rerank_scores(const float *states, uint32_t n, uint32_t hidden, const float *pooler_weight,
                                 const float *pooler_bias, const float *classifier_weight, float classifier_bias,
                                 float *scores, turbo_error *err);

/* turbo_rocm_rerank_run: the windows of `pairs` pairs ([windows, seq] ids and
 * types, each window's length, and the pair it belongs to) through a
 * TURBO_TASK_RERANK session of this backend, max_batch windows a run, as
 * CLS rows at full width with no normalization, then the head above, computed
 * on the device with its tensors copied there on every call (the same F64
 * products; the classifier's sum in another order, so a score may be an F32
 * rounding off the host's); each pair's score is the largest of its windows'
 * (core/src/session/rerank.rs:111-219). pairs may not exceed the session's
 * max_batch. */
int32_t turbo_rocm_rerank_run(void *session, const int32_t *ids, const int32_t *types, const uint32_t *lengths,
                              uint32_t windows, uint32_t seq, const uint32_t *owner, uint32_t pairs,
                              const float *pooler_weight, const float *pooler_bias, const float *classifier_weight,
                              float classifier_bias, float *scores, turbo_error *err);

/* turbo_rocm_buffer_quantize_static: this backend's buffer_quantize entry
 * without an allocation. It has no counterpart in the reference: it is for
 * callers that cannot allocate device memory (code under HIP graph capture,
 * tight serving loops, harnesses that forbid hipMalloc). The same codes, byte
 * for byte, as buffer_quantize, staged in a fixed device area of 16 MiB a GPU
 * (allocated once with the library, held until the process ends) instead of
 * memory allocated per call: the codes, then on a 256-byte boundary the int8
 * ranges ([2, dim] F32), must fit it, or the call fails with
 * TURBO_E_INVALID_ARGUMENT before any device work. It calls no allocating
 * routine. Every context on a GPU shares that GPU's area; a lock per GPU,
 * held through the call, serializes calls from any thread and context. run,
 * when not NULL, gets the int8 ranges' bytes in h2d_bytes and the device
 * allocations the call made (none) in device_allocs. */
int32_t turbo_rocm_buffer_quantize_static(void *buffer, uint32_t quantization, const float *int8_ranges, uint32_t rows,
                                          uint32_t dim, turbo_backend_run *run, turbo_error *err);

/* ---- Operators on device memory (no counterpart in the reference) ----
 *
 * What a program needs to run layers of its own over a session's states
 * (taps, hidden states, imported embeddings): an RMS norm with the residual's
 * addition and int8 codes out, those codes of any rows, the int8 product on
 * codes and scales, and the attention of its tokens to an encoder's states of
 * another length. Like buffer_quantize they work on memory that the caller
 * owns.
 *
 * Each takes a context and a call struct whose first field is struct_size
 * (another size: TURBO_E_INVALID_STRUCT_SIZE). Every argument is checked on
 * the host before any device work (those that a NULL context could serve
 * first, then the context: TURBO_E_INVALID_HANDLE); a refused call has written
 * nothing, and its error's field is the place, from 1, of the array it is
 * about among the call's arrays, or 0. With
 * TURBO_ROCM_ENQUEUE in flags the kernels are enqueued on `stream` (a
 * hipStream_t of the context's device; NULL: that device's default stream)
 * and the call returns: it allocates nothing, waits for nothing and may be
 * captured into a graph. A stream of another device is refused. Without the
 * flag `stream` must be NULL, and the call runs on the context's own stream
 * and returns when its results are there. Calls
 * keep no state of their own: any number may run at once, from any threads
 * and on any streams, when none writes memory that another reads or writes.
 * The calling thread's current device may be any; it is the caller's again
 * afterwards. */
#define TURBO_ROCM_ENQUEUE 1u

/* HIP's number of a context's device (the table's ordinals count the devices
 * that the backend lists), for a caller to see where an array has to be. */
int32_t turbo_rocm_context_device(void *ctx, uint32_t *device, turbo_error *err);

/* An array in device-addressable memory: `data` is the address of its first
 * element on the context's device (a buffer's exported
 * TURBO_HANDLE_CUDA_PTR, or any memory of that device), and `bytes` what lies
 * behind it there. ndim 1 to 3; the last axis is contiguous, stride[i] is the
 * elements from one step of axis i to the next (for i < ndim - 1; the other
 * strides are ignored). Strides need not keep an order and 0 repeats an input;
 * an output's elements must not overlap. Every element is checked to lie
 * within `bytes`; data must be aligned to one element. An absent optional
 * array is all zeros (ndim 0). An array with an empty axis is never read, and
 * its data may be NULL. */
typedef struct turbo_rocm_tensor {
    void    *data;
    uint64_t bytes;
    uint64_t shape[3];
    uint64_t stride[2];
    uint32_t ndim;
    uint32_t dtype;   /* TURBO_DTYPE_* */
} turbo_rocm_tensor;

/* turbo_rocm_rms_norm: rows of `cols` values, at most 65536. For each row
 *
 *   v = x, or x + residual in F32 rounded once to the residual's type
 *   y = v * weight / sqrt(mean(v^2) + eps)      (64-bit sums and products)
 *
 * x [rows, cols] F32, F16 or BF16; residual [rows, cols] (optional) of x's
 * type or F32; weight [cols], F32 or x's type; eps positive and finite.
 * Outputs, any of:
 *   sum [rows, cols], the residual's type: v (only with a residual). It may
 *     be the residual itself, or x where the types are equal: same address
 *     and strides.
 *   out [rows, cols], F32, F16 or BF16: y, rounded once (BF16 below F32's
 *     smallest normal number: to F32 first). It may be x, in the same way.
 *   codes [rows, cols] I8 with scales [rows] F32: symmetric int8 codes of y's
 *     row before any rounding: scale = max|y| / 127 rounded to F32, code =
 *     the whole number nearest to 127 y / max|y|, ties to even, exactly. A row
 *     of zeros has scale 0 and codes 0. A row with an infinity or NaN among
 *     its v * weight has scale NaN and codes 0, so whatever reads the codes
 *     sees it.
 * One of out and codes at least; sum, out and codes may not overlap each
 * other, nor an input except as said. */
typedef struct turbo_rocm_rms_norm_call {
    uint32_t struct_size;
    uint32_t flags;
    void    *stream;
    double   eps;
    turbo_rocm_tensor x, residual, weight, sum, out, codes, scales;
} turbo_rocm_rms_norm_call;
int32_t turbo_rocm_rms_norm(void *ctx, const turbo_rocm_rms_norm_call *call, turbo_error *err);

/* turbo_rocm_quantize_tokens: the codes and scales above of the rows of x
 * [rows, cols] (F32, F16 or BF16; at most 65536 columns) themselves, as an
 * int8 product takes them. */
typedef struct turbo_rocm_quantize_tokens_call {
    uint32_t struct_size;
    uint32_t flags;
    void    *stream;
    turbo_rocm_tensor x, codes, scales;
} turbo_rocm_quantize_tokens_call;
int32_t turbo_rocm_quantize_tokens(void *ctx, const turbo_rocm_quantize_tokens_call *call, turbo_error *err);

/* turbo_rocm_linear_i8: out[m, n] = (sum_k codes[m, k] weight[n, k]) *
 * scales[m] * weight_scales[n] + bias[n], the sum exact in 32-bit integers
 * (inner width at most 131071, where the largest sum still fits), the rest in
 * F32 (the sum, its product with scales[m] and the multiply-add with the bias
 * round there), rounded once to out's type. codes [M, K] and weight [N, K] I8, scales
 * [M], weight_scales [N] and bias [N] (optional) F32, out [M, N] F32, F16 or
 * BF16. K 0 gives the bias (or zeros, as an empty sum times the scales). out
 * may not overlap an input. */
typedef struct turbo_rocm_linear_i8_call {
    uint32_t struct_size;
    uint32_t flags;
    void    *stream;
    turbo_rocm_tensor codes, scales, weight, weight_scales, bias, out;
} turbo_rocm_linear_i8_call;
int32_t turbo_rocm_linear_i8(void *ctx, const turbo_rocm_linear_i8_call *call, turbo_error *err);

/* Cross attention: the queries of each sequence attend to the encoder states
 * of that sequence, whose number is another. Sequences are packed one after
 * another: sequence s has q_lens[s] query tokens behind those of the
 * sequences before it, and k_lens[s] states likewise (both host arrays of
 * `batch`; 0 is allowed). Query head h reads key and value head h / (heads /
 * kv_heads); heads must be a multiple of kv_heads. width is the head width, 1
 * to 128. dtype F32, F16 or BF16.
 *
 * turbo_rocm_cross_plan_create works out, for these lengths on the context's
 * device, which workgroup takes which tokens and keys, and keeps that on the
 * device. A plan is never written after that: one serves any number of calls
 * (a decoder's layers and steps) on any streams, at once. It must outlive the
 * calls and graphs that use it, and its context the calls.
 * *workspace_bytes (may be NULL) is what each call needs beside its operands.
 * More than 2^31 rows (query tokens times heads) or states, or 2^23
 * workgroups, are TURBO_E_CAPACITY. */
typedef struct turbo_rocm_cross_desc {
    uint32_t struct_size;
    uint32_t dtype;
    uint32_t batch;
    uint32_t heads;
    uint32_t kv_heads;
    uint32_t width;
    const uint32_t *q_lens;
    const uint32_t *k_lens;
} turbo_rocm_cross_desc;
int32_t turbo_rocm_cross_plan_create(void *ctx, const turbo_rocm_cross_desc *desc, uint64_t *workspace_bytes,
                                     void **out, turbo_error *err);
void turbo_rocm_cross_plan_release(void *plan);

/* turbo_rocm_cross_attention: for each query token i and head h of a sequence
 *
 *   out[i, h] = sum_j p_j v[j, h'],  p = softmax over j of scale * q[i, h] . k[j, h']
 *
 * over the sequence's live states j; h' is the head that h reads. q and out
 * [tokens, heads, width], k and v [states, kv_heads, width], in the plan's
 * type, with at least the plan's tokens and states (out's rows past the last
 * sequence are left as they were). mask [states] I32 (optional): a state whose
 * entry is 0 is not live, and nothing of its key and value is used, whatever
 * they hold. A query with no live state has a zero output. scale finite in F32.
 * Scores, probabilities and sums are F32; 16-bit operands round a probability
 * for the product with V, to their type or, in calls of few rows, to the sum of
 * two numbers of it, and the output once. Values are summed with weights of at
 * most 1 (256 for F16) and divided at the end: outputs are finite where the
 * largest |v| times the number of live states is, in F32. A score of plus
 * infinity or one that is undefined gives what the formula gives, a NaN; one of
 * minus infinity weighs nothing. workspace: `workspace_bytes` of the context's
 * device, 16-byte aligned, at least the plan's, for this call alone until it has
 * finished (two graphs that may run at once need one each). It holds nothing
 * between calls. out may not overlap an input or the workspace. */
typedef struct turbo_rocm_cross_attention_call {
    uint32_t struct_size;
    uint32_t flags;
    void    *stream;
    void    *workspace;
    uint64_t workspace_bytes;
    double   scale;
    turbo_rocm_tensor q, k, v, mask, out;
} turbo_rocm_cross_attention_call;
int32_t turbo_rocm_cross_attention(void *plan, const turbo_rocm_cross_attention_call *call, turbo_error *err);

/* The checks of a plan's description and of a call with it, as the two
 * functions above make them (but for the workspace, which the plan sizes),
 * without a device; call may be NULL. */
int32_t turbo_rocm_cross_check(const turbo_rocm_cross_desc *desc, const turbo_rocm_cross_attention_call *call,
                               turbo_error *err);

/* ---- Test and measurement hooks (no counterpart in the reference's seam; the
 * reference's CUDA backend keeps similar ones, core/src/cuda.rs:177-499) ---- */

/* Makes the GEMM block shape `name` (as a choices string spells it, e.g.
 * "256x256"; NULL or "" for none) fail to launch from now on, in place of a
 * device that cannot take it: the launcher's rule picks another shape, the
 * tuner skips it, a cached choice naming it is not taken, and a session that
 * forces it is refused with TURBO_E_UNSUPPORTED (the reference's
 * turbo_cuda_fail_variant, core/src/cuda.rs:461-469,
 * core/cuda/backend.cpp:2430-2440, 3006-3010). Process-wide. */
int32_t turbo_rocm_fail_variant(const char *name, turbo_error *err);

/* Which kernel turbo_rocm_linear_i8 runs for [m, k] codes by [n, k] weights,
 * without a device: 0 for k below 16, 1 to 4 for pieces of so many 16 rows, 64,
 * 128 or 256 for tiles of that edge (a product of more than 2^22 64 x 64 tiles
 * goes by halves, each with its own). aligned: both operands' addresses and
 * strides, and k, are multiples of 16. */
int32_t turbo_rocm_linear_i8_kernel(uint32_t m, uint32_t n, uint32_t k, uint32_t aligned, uint32_t *kernel,
                                    turbo_error *err);

/* How a cross attention plan of this description is cut, without a device: the
 * most rows (query tokens' heads that read one key head) of a workgroup, 32 or
 * 128, and the most states; a sequence of more states is joined from parts. */
int32_t turbo_rocm_cross_cut(const turbo_rocm_cross_desc *desc, uint32_t *rows, uint64_t *states, turbo_error *err);

/* The last run's packing, read back from the device: each row's first packed
 * token and length ([batch] each), each packed token's r * seq + p ([tokens]),
 * and the packed token count. */
int32_t turbo_rocm_session_packing(void *session, int32_t *start, int32_t *len, int32_t *at, uint32_t *tokens,
                                   turbo_error *err);

/* The last run's final hidden states, [tokens, hidden] F32. */
int32_t turbo_rocm_session_hidden(void *session, float *out, uint64_t floats, turbo_error *err);

/* The backend's heap allocations so far: every malloc-family and operator
 * new call its own code has made (counted as they happen), in the process
 * and on the calling thread. A run's turbo_backend_run.host_allocs is the
 * change of the thread's count across it. Either pointer may be NULL. */
int32_t turbo_rocm_host_allocs(uint64_t *process, uint64_t *thread, turbo_error *err);

/* Times every kernel of the session's later runs with HIP events, each
 * launch's pair bound to its kernels' own dispatch packets (the first
 * kernel's start, the last one's end: no marker packet between launches) on
 * the stream it runs on (a split run's parts side by side, as the run
 * executes them; timed runs launch their kernels directly rather than
 * replay a graph, and take a replay's time); turbo_rocm_session_times then writes
 * "<kernel> <ms> <launches>" lines: the milliseconds summed over the last
 * run's launches of that kernel, and how many there were;
 * turbo_rocm_session_intervals writes "<kernel> <start> <end>" a launch, in
 * ms from the run's start, in launch order. */
int32_t turbo_rocm_session_timing(void *session, uint32_t on, turbo_error *err);
int32_t turbo_rocm_session_times(void *session, char *out, uint32_t len, turbo_error *err);
int32_t turbo_rocm_session_intervals(void *session, char *out, uint32_t len, turbo_error *err);

/* Runs the last written rows `runs` more times, back to back on the
 * context's stream, then waits: the rows stay resident on the device, so
 * this is the device's throughput on them, for measurement. */
int32_t turbo_rocm_session_replay(void *session, uint32_t runs, turbo_error *err);

/* How many graphs the session has captured (one per bin of packed tokens, at
 * session_open) and how many runs replayed one since. */
int32_t turbo_rocm_session_graphs(void *session, uint64_t *captured, uint64_t *launched, turbo_error *err);

/* The session's kernel choices, as TURBO_ROCM_CHOICES takes them. */
int32_t turbo_rocm_session_choices(void *session, char *out, uint32_t len, turbo_error *err);

/* One GEMM, out [M, N] = A [M, K] W [N, K]^T + bias (bias may be NULL), with
 * the operands narrowed on the device to dtype (TURBO_DTYPE_F32, F16 or
 * BF16) or quantized to int8 rows (TURBO_DTYPE_I8: a symmetric scale per row
 * of A and of W, int32 sums, dequantized in F32), and block shape `tile`
 * (0 = the default choice). Allocates its own device memory; for kernel tests. */
int32_t turbo_rocm_gemm_check(uint32_t ordinal, uint32_t dtype, uint32_t M, uint32_t N, uint32_t K, const float *A,
                              const float *W, const float *bias, float *out, uint32_t tile, turbo_error *err);

/* The average milliseconds of `iters` back-to-back launches of the GEMM
 * [M, K] x [N, K]^T with the residual epilogue, block shape `tile`, on
 * device-resident uniform random operands of dtype; for tuning sweeps. */
int32_t turbo_rocm_gemm_time(uint32_t ordinal, uint32_t dtype, uint32_t M, uint32_t N, uint32_t K, uint32_t tile,
                             uint32_t iters, float *ms, turbo_error *err);

/* A plain device copy of `bytes` (a multiple of 16) from one buffer to
 * another, `iters` times, on device `ordinal`: the average milliseconds of
 * a launch into *ms. A measurement hook with no counterpart
 * in the reference: its launches read and write exactly `bytes`, so the
 * profiler's traffic counters can be scaled by what they read for it. */
int32_t turbo_rocm_copy_probe(uint32_t ordinal, uint64_t bytes, uint32_t iters, float *ms, turbo_error *err);

/* The matrix cores' sustained rate: every compute unit's 4 waves issue 8
 * independent chains of 32x32x16 F16 products for iters rounds, with fixed
 * operands, or with random ones changing every product (random 1), as a
 * GEMM's do; *tflops is the rate, *mhz the shader clock under that load. A
 * measurement hook with no counterpart in the reference: the ceiling a
 * GEMM's data lets the chip sustain, beside the published peak. */
int32_t turbo_rocm_mfma_probe(uint32_t ordinal, uint32_t random, uint32_t iters, float *tflops, float *mhz,
                              turbo_error *err);

#ifdef __cplusplus
}
#endif

#endif /* TURBO_ROCM_H */
