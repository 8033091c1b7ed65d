/*
 * motifcl_amd.h -- C ABI of the MI355X (gfx950) compact-counter update library.
 *
 * Every entry point takes plain device pointers with their byte sizes, scalar
 * arguments and a HIP stream (hipStream_t passed as void*, NULL = the default
 * stream).  Work is enqueued on that stream and the call returns without
 * waiting.  Return value: 0 (MCC_OK) on success, a negative MCC_E_* code on
 * failure; mcc_last_error() then returns the message for the calling thread.
 * Validation failures never enqueue work and never throw -- the convention of
 * the reference's VulkanOpResult{success,error}
 * (include/motifcl/runtime/vulkan_backend.hpp:80-84).
 *
 * Data layout (kernels/compact_counter.cl:1-5):
 *   state  u8  [out, in/4, 3]  four 6-bit codes per 3 bytes, little-endian
 *                              24-bit word c0 | c1<<6 | c2<<12 | c3<<18
 *   scale  f32 [out]           per-row weight scale
 *   v      f32 [out]           per-row RMS second moment
 *   grad_w f32 [out, in]       dense weight gradient, row-major
 *   x      f32 [batch, in]     layer input, row-major
 *   grad_out f32 [batch, out]  upstream gradient, row-major
 */
#ifndef MOTIFCL_AMD_H
#define MOTIFCL_AMD_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define MCC_OK 0
#define MCC_E_INVALID (-1) /* argument validation failed; nothing was enqueued */
#define MCC_E_RUNTIME (-2) /* a HIP call failed */

/* Message of the last failure on this thread ("" if none). */
const char* mcc_last_error(void);

/* Name and architecture of the current HIP device, e.g. "AMD Instinct MI355X (gfx950)".
 * Replaces VulkanOpResult::device_name. */
const char* mcc_device_name(void);

/*
 * Update-only step: the optimizer step for a supplied dense weight gradient.
 * Replaces CounterStateLinear::apply_update_seed
 * (src/nn/compact_counter.cpp:113-156: counter_row_stats_f32 ->
 * counter_apply_update_f32 -> copy_f32; kernels/compact_counter.cl:59-139).
 * Mutates state, scale and v in place.  Results are bit-identical to the
 * reference arithmetic evaluated in IEEE-754 binary32 without contraction.
 */
int mcc_compact_counter_apply_update_dense(
    void* stream,
    uint8_t* state, size_t state_nbytes,
    float* scale, size_t scale_nbytes,
    float* v, size_t v_nbytes,
    const float* grad_w, size_t grad_w_nbytes,
    size_t C, size_t in_features, size_t out_features,
    float lr, float lr_scale, float rms_beta, float rms_eps, uint32_t seed);

/*
 * Update-only step for a list of counter tensors in one call -- the optimizer step of a
 * whole model when every dense weight gradient is already in memory.  Each tensor gets
 * exactly the result of mcc_compact_counter_apply_update_dense with its own lr and seed;
 * C, lr_scale, rms_beta and rms_eps are shared.  The reference applies the update layer by
 * layer from the host (CounterStateLinear::apply_update_seed,
 * src/nn/compact_counter.cpp:113-156, once per module; the layer lists it walks are e.g.
 * tools/train_ternary15m.cpp:313-318); one launch over the rows of many tensors keeps the
 * memory system and the ALUs busy together, which a single small tensor cannot.
 * `tensors` is a host array; tensors must not alias each other.
 */
typedef struct mcc_counter_tensor {
    uint8_t* state;      size_t state_nbytes;
    float* scale;        size_t scale_nbytes;
    float* v;            size_t v_nbytes;
    const float* grad_w; size_t grad_w_nbytes;
    size_t in_features, out_features;
    float lr;
    uint32_t seed;
} mcc_counter_tensor;

int mcc_compact_counter_apply_update_dense_batched(
    void* stream, const mcc_counter_tensor* tensors, size_t n_tensors,
    size_t C, float lr_scale, float rms_beta, float rms_eps);

/*
 * Bytes of transient workspace mcc_compact_counter_apply_update_fused needs
 * for the given shape (0 on invalid dimensions): out*in*4 times the number of
 * token chunks the contraction is split into, plus 1 KiB of hand-off words
 * for large shapes that are not a whole number of rounds of 256 x 256 tiles
 * (their contraction then runs as one launch of equal spans; a workspace of
 * out*in*4 bytes without the words is accepted and gives the same bytes).
 * Layers with fewer than about 1024 output tiles split their tokens so that
 * the whole GPU works on them; the size depends on (in, out, batch) only.
 */
size_t mcc_compact_counter_fused_workspace_nbytes(size_t in_features, size_t out_features,
                                                  size_t batch);

/*
 * Bytes of the small workspace with which mcc_compact_counter_apply_update_fused
 * runs without a buffer of the size of the weight gradient, or 0 when the shape
 * has no way smaller than the full workspace (tiny layers).  Layers whose in and
 * out are multiples of 128 with in >= 768 take the accumulator-resident strip
 * path: 512 bytes of partial row sums per output row plus a few control words,
 * and, for layers of more than 256 tiles of 256 x 256, room to park 2 (in/256 - 1)
 * such tiles between the passes of the kernel's grid (24 MB for the largest layer
 * of a 7B model instead of 180 MB).  Every other shape
 * is updated band by band of an eighth of its output rows: the workspace holds
 * one band's gradient.  No counterpart in the reference, whose fused kernels
 * recompute the gradient instead of holding it.
 */
size_t mcc_compact_counter_fused_strip_workspace_nbytes(size_t in_features, size_t out_features,
                                                        size_t batch);

/*
 * Waits for `stream` and reports whether every strip-path step of this process
 * on the current GPU since the last call completed: MCC_OK, or MCC_E_RUNTIME
 * when a step gave up a wait between tiles.  Such a step leaves whole strips
 * (128 or 256 rows) of its tensor without their update -- state, scale and v of those rows
 * are untouched, no strip is half-updated -- and the report clears the count.
 * The count lives in the library, per GPU, so it survives other layers' steps
 * through the same workspace; the workspace and shape arguments are not looked
 * at (kept for callers written against the first form of this call).  Always
 * MCC_OK for steps on the full workspace or band by band.  No counterpart in
 * the reference.
 */
int mcc_compact_counter_fused_check(void* stream, const void* workspace, size_t workspace_nbytes,
                                    size_t in_features, size_t out_features, size_t batch);

/*
 * Fused step: weight-gradient contraction grad_w = grad_out^T . x on the fp32
 * matrix cores followed by the counter update.
 * Replaces run_vulkan_compact_counter_apply_update_fused
 * (include/motifcl/runtime/vulkan_backend.hpp:733-749,
 *  src/runtime/vulkan_backend.cpp:8475-8578) and the OpenCL twin in
 * CounterStateLinear::apply_update_backward (src/nn/compact_counter.cpp:158-231).
 * The reference's scale_new/denom scratch buffers are not needed; instead the
 * caller lends `workspace`, whose size selects how the step runs:
 *   - >= mcc_compact_counter_fused_workspace_nbytes (one f32[out,in] slice
 *     per token chunk of the contraction; large layers have one chunk):
 *     contraction into the workspace, then the update kernel.  After the call
 *     the first out*in floats of the workspace hold grad_w.  The fastest way.
 *   - >= mcc_compact_counter_fused_strip_workspace_nbytes but smaller than
 *     the above: no weight-sized buffer exists at any time, which is the
 *     property tests/test_memory_truth_gate.cpp:109-113 of the reference asks
 *     for.  Any lr_scale.  On the strip path (see the size query) the update is
 *     applied from the contraction's accumulators; x must be 16-byte aligned;
 *     tiles of one row strip wait for each other on the device, so two such
 *     steps must not run side by side on one GPU: a call on another stream than
 *     the previous strip call is ordered behind it on the device (the stream
 *     waits for an event recorded after that call; the host does not wait),
 *     every wait is bounded, and mcc_compact_counter_fused_check reports a
 *     wait that was given up.  On a stream under graph capture no such order
 *     is added: do not replay two such graphs side by side.
 * The ways produce identical bytes whenever none of them splits the tokens into
 * chunks, i.e. for fewer than 512 tokens or layers of at least 1024 tiles of
 * 128 x 128 (mcc_compact_counter_fused_workspace_nbytes == out*in*4); where
 * one does, its gradient is the sum of chunk sums and they differ by that
 * rounding (a few counters in 10^5 flip differently).
 * grad_w differs from the reference's
 * sequential fp32 sum only by summation order (relative error <= 1e-4 of the
 * row norm); given that grad_w the counter arithmetic is the same as in the
 * dense entry point.
 */
int mcc_compact_counter_apply_update_fused(
    void* stream,
    uint8_t* state, size_t state_nbytes,
    float* scale, size_t scale_nbytes,
    float* v, size_t v_nbytes,
    const float* grad_out, size_t grad_out_nbytes,
    const float* x, size_t x_nbytes,
    void* workspace, size_t workspace_nbytes,
    size_t C, size_t in_features, size_t out_features, size_t batch,
    float lr, float lr_scale, float rms_beta, float rms_eps, uint32_t seed);

/*
 * The fused step with the workspace inside the library: the same step as
 * mcc_compact_counter_apply_update_fused, for callers that cannot allocate device
 * memory -- code under HIP graph capture, tight serving loops, harnesses that
 * forbid hipMalloc.  It has no counterpart in the reference.  The workspace is a
 * static device array of MCC_NOALLOC_WORKSPACE_NBYTES bytes that every GPU the
 * library runs on holds from its first use there until the process ends; the
 * call itself allocates nothing (no hipMalloc / hipFree, no stream-ordered
 * allocation; with mcc_profiler_enable(1) the profiler may still create events).
 * The step runs as mcc_compact_counter_apply_update_fused would with
 *   - mcc_compact_counter_fused_workspace_nbytes(in, out, batch) bytes when that
 *     fits the array (identical bytes to that call), else
 *   - mcc_compact_counter_fused_strip_workspace_nbytes(in, out, batch) bytes when
 *     that fits, else
 *   - it fails with MCC_E_INVALID and a message that names both sizes.
 * All calls on one GPU share that GPU's array, which keeps the last call's
 * contents: two calls that overlap in time on one GPU (different streams) race.
 * The first call on a GPU looks up the array's address there (and, for a shape
 * on the strip path, creates the event that orders strip steps of different
 * streams): make that first call outside graph capture; later calls may be
 * captured and replayed.  A step that took the strip path reports a given-up
 * wait through mcc_compact_counter_fused_check, like the lent-workspace call
 * (its workspace arguments are not looked at: pass a null pointer and 0).
 * Arguments and validation are those of mcc_compact_counter_apply_update_fused
 * without the workspace.
 */
#define MCC_NOALLOC_WORKSPACE_NBYTES ((size_t)32 << 20)
int mcc_compact_counter_apply_update_fused_static(
    void* stream,
    uint8_t* state, size_t state_nbytes,
    float* scale, size_t scale_nbytes,
    float* v, size_t v_nbytes,
    const float* grad_out, size_t grad_out_nbytes,
    const float* x, size_t x_nbytes,
    size_t C, size_t in_features, size_t out_features, size_t batch,
    float lr, float lr_scale, float rms_beta, float rms_eps, uint32_t seed);

/*
 * The fused step for a list of tensors in a handful of launches: one grouped
 * contraction per tile size, one launch that adds the token-chunk slices, and
 * the batched update.  For models made of small layers (the 288- and 768-wide
 * linears of the 15M-parameter model) the per-tensor entry point is bound by
 * its three launches per tensor; this one costs about five launches for all of
 * them.  It has no single counterpart in the reference: it stands for the
 * per-layer calls of apply_update_backward (src/nn/compact_counter.cpp:158-231)
 * of a caller that keeps every layer's grad_out and x alive until the end of
 * its backward pass, which is equivalent because no layer's update reads
 * another layer's state.  state, scale and v come out bit-identical to calling
 * mcc_compact_counter_apply_update_fused per tensor with a full workspace --
 * except for a list that runs as equal spans: when every layer's sides are
 * multiples of 256, every token count a multiple of 16 and the list holds at
 * least 512 tiles of 256 x 256 (the 110M-shaped model: 1296), the contractions
 * of the whole list are one launch in which every workgroup gets an equal share
 * of the list's tiles and tokens, with no token chunks: each gradient is then
 * the unchunked token-order sum (the reference's order up to pairing), state,
 * scale and v are exact for that gradient, and they equal the per-tensor call's
 * wherever that call does not split the tokens into chunks and differ from it
 * by the rounding of its chunk sums elsewhere (counter-flip fraction ~1e-6).
 * Such a list needs 16-byte aligned grad_out and x.
 * Likewise a list of small layers whose tiles together number 512 or more (the
 * 15M-shaped model: 42 layers) is cut into token chunks per list, fewer than a
 * layer's own call would use: its gradients are the sums over those chunks,
 * state, scale and v exact for them, with the same relation to the per-tensor
 * call.
 * `workspace` (256-byte aligned) holds
 * mcc_compact_counter_fused_batched_workspace_nbytes(tensors, n) bytes: the
 * per-tensor workspaces, each rounded up to 256 bytes, one after the other (as
 * equal spans: out * in floats per tensor plus 1 KiB; the size depends on the
 * calling thread's contraction mode, so query it in the mode the call runs in).
 * Under MCC_CONTRACTION_BF16X6 the tensors are processed one by one.
 */
typedef struct mcc_fused_tensor {
    uint8_t* state;        size_t state_nbytes;
    float* scale;          size_t scale_nbytes;
    float* v;              size_t v_nbytes;
    const float* grad_out; size_t grad_out_nbytes;  /* [batch, out_features] */
    const float* x;        size_t x_nbytes;         /* [batch, in_features] */
    size_t in_features, out_features, batch;
    float lr;
    uint32_t seed;
} mcc_fused_tensor;
size_t mcc_compact_counter_fused_batched_workspace_nbytes(const mcc_fused_tensor* tensors, size_t n_tensors);
int mcc_compact_counter_apply_update_fused_batched(
    void* stream, const mcc_fused_tensor* tensors, size_t n_tensors,
    void* workspace, size_t workspace_nbytes,
    size_t C, float lr_scale, float rms_beta, float rms_eps);

/*
 * How the weight-gradient contraction (inside the two-kernel fused step and in
 * mcc_matmul_transpose_a_f32) multiplies.  A setting of the calling thread: it
 * governs the calls that thread makes afterwards and no other thread's.  No
 * counterpart in the reference.
 *   MCC_CONTRACTION_FP32    the fp32 matrix instruction (default)
 *   MCC_CONTRACTION_BF16X6  both operands split into three bf16 terms, six bf16
 *                           matrix passes per product: per-product error of one
 *                           binary32 rounding, as the fp32 instruction, at about
 *                           1.2 x its speed on 7B-sized layers (72 against 88 ms
 *                           for a seven-tensor layer step at 32768 tokens).  Used
 *                           for whole 128 x 128 tiles and
 *                           token counts that are multiples of 32; other shapes
 *                           silently use the fp32 instruction.  The two modes give
 *                           gradients that differ in the last bits, so counters
 *                           whose tick lands within that distance of a rounding
 *                           boundary may come out differently.
 */
#define MCC_CONTRACTION_FP32 0
#define MCC_CONTRACTION_BF16X6 1
int mcc_set_contraction_mode(int mode);
int mcc_get_contraction_mode(void);

/*
 * c[m,n] = a[k,m]^T . b[k,n], fp32, row-major.
 * Replaces matmul_transpose_a (include/motifcl/ops/matmul.hpp:8,
 * src/ops/matmul.cpp:1416-1418), the producer of the dense weight gradient
 * (grad_w = matmul_transpose_a(grad_out, x), tests/test_memory_truth_gate.cpp:49).
 */
int mcc_matmul_transpose_a_f32(
    void* stream,
    const float* a, size_t a_nbytes,
    const float* b, size_t b_nbytes,
    float* c, size_t c_nbytes,
    size_t k, size_t m, size_t n);

/*
 * weight[out,in] = scale[row] * t(state).
 * Replaces run_vulkan_compact_counter_decode_weight
 * (include/motifcl/runtime/vulkan_backend.hpp:713-719,
 *  src/runtime/vulkan_backend.cpp:8603-8660; kernels/compact_counter.cl:39-55).
 */
int mcc_compact_counter_decode_weight(
    void* stream,
    const uint8_t* state, size_t state_nbytes,
    const float* scale, size_t scale_nbytes,
    float* weight, size_t weight_nbytes,
    size_t in_features, size_t out_features, size_t C);

/*
 * out[batch,out] = x[batch,in] . W(state)^T with the ternary weights decoded
 * from the packed state inside the contraction (no dense weight buffer).
 * Runs on the bf16 matrix cores with every product exact: the ternary weight
 * is exact in bf16 and each activation is split into three bf16 terms whose sum
 * is the activation, so the result has fp32 accuracy (the terms of an fp32
 * contraction, summed in another order).  Activations must be finite and
 * below 3.38e38 in magnitude (the largest bf16); terms below 2^-110 lose
 * their low bits.
 * Replaces run_vulkan_compact_counter_forward_u8
 * (include/motifcl/runtime/vulkan_backend.hpp:722-730,
 *  src/runtime/vulkan_backend.cpp:8662-8725).
 */
int mcc_compact_counter_forward_u8(
    void* stream,
    const float* x, size_t x_nbytes,
    const uint8_t* state, size_t state_nbytes,
    const float* scale, size_t scale_nbytes,
    float* out, size_t out_nbytes,
    size_t batch, size_t in_features, size_t out_features, size_t C);

/*
 * grad_x[batch,in] = grad_out[batch,out] . W(state), decoded in-kernel; grad_out
 * is multiplied by the row scale first, as the reference does, then split as in
 * the forward product (same accuracy, same requirement of finite inputs).
 * Replaces run_vulkan_compact_counter_backward_input_u8
 * (include/motifcl/runtime/vulkan_backend.hpp:750-758,
 *  src/runtime/vulkan_backend.cpp:8727-8803; kernels/compact_counter.cl:248-269).
 */
int mcc_compact_counter_backward_input_u8(
    void* stream,
    const uint8_t* state, size_t state_nbytes,
    const float* scale, size_t scale_nbytes,
    const float* grad_out, size_t grad_out_nbytes,
    float* grad_x, size_t grad_x_nbytes,
    size_t batch, size_t in_features, size_t out_features, size_t C);

/*
 * FP32 side optimizers for the non-counter tensors of a counter model
 * (embedding, norm gains).  Replace sgd_update and adam_update_fast
 * (include/motifcl/ops/optim.hpp, src/ops/optim.cpp:17-86; kernels
 * kernels/optim.cl:1-7,31-53).  `n` counts elements; all buffers hold n floats.
 * Adam: step >= 1; the bias corrections 1/(1 - beta^step) are computed on the
 * host in binary32 as the reference does (src/ops/optim.cpp:70-71).
 */
int mcc_sgd_update_f32(void* stream, float* param, size_t param_nbytes, const float* grad,
                       size_t grad_nbytes, size_t n, float lr);
int mcc_adam_update_f32(void* stream, float* param, size_t param_nbytes, const float* grad,
                        size_t grad_nbytes, float* m, size_t m_nbytes, float* v, size_t v_nbytes,
                        size_t n, float lr, float beta1, float beta2, float eps, int step,
                        float weight_decay);

/*
 * Row-wise operators around the counter layers: the norm in front of them, whose gain and bias the side
 * optimizers train, and the log probabilities and the distillation loss behind the vocabulary head,
 * whose gradient starts the backward pass.  The reference has a norm and a loss of its own among its
 * general ops (src/ops/norm.cpp, src/ops/loss.cpp); these are no replacements of them call by call.
 *
 * Large tensors are rows of elements of one type, MCC_ELEMENT_*, aligned to the element; a stride counts
 * the elements from the start of a row to that of the next (at least the row's length).  Whatever the
 * type, everything is computed in binary32 (sums whose error would grow with the length of a row or the
 * number of rows in binary64) and a result is rounded to the type once.  An output may replace an input of
 * the same type where that is said (same pointer, same stride); any other overlap of the large tensors is
 * refused.  Equal calls give equal bytes.  Rows hold at most 2^30 elements.
 * Nothing is allocated and nothing is kept between calls: all entry points may be captured into a graph.
 * Workspaces are aligned to 16 bytes and belong to the call until it has run; their sizes depend on the
 * arguments of the query alone and may be 0 (then the pointer may be null).
 */
#define MCC_ELEMENT_F32 0
#define MCC_ELEMENT_F16 1
#define MCC_ELEMENT_BF16 2

/*
 * y = (x - mean) * rstd * gain + bias with the row's mean and rstd = 1 / sqrt(variance + eps), the
 * variance being the mean of the squared differences.  gain and bias (cols floats) may be null: 1 and 0.
 * mean and rstd (rows floats), which the backward pass needs, may be null.  y may replace x.  Squared
 * differences have to lie in the range of binary32: beyond 2^64 from the mean rstd is 0 and y the bias.
 */
int mcc_layer_norm(void* stream, const void* x, size_t x_nbytes, size_t x_stride, const float* gain, size_t gain_nbytes,
                   const float* bias, size_t bias_nbytes, void* y, size_t y_nbytes, size_t y_stride, float* mean,
                   size_t mean_nbytes, float* rstd, size_t rstd_nbytes, size_t rows, size_t cols, int element, float eps);

/*
 * Gradients of x, gain and bias for grad_out, the gradient of y, with the mean and rstd of the forward
 * call.  grad_x, grad_gain and grad_bias may be null (not wanted); gain as in the forward call.  grad_x
 * may replace grad_out or x.  grad_gain and grad_bias (cols floats) are overwritten with the sums over
 * all rows.
 */
size_t mcc_layer_norm_backward_workspace_nbytes(size_t rows, size_t cols, int element);
int mcc_layer_norm_backward(void* stream, const void* grad_out, size_t grad_out_nbytes, size_t grad_out_stride,
                            const void* x, size_t x_nbytes, size_t x_stride, const float* mean, size_t mean_nbytes,
                            const float* rstd, size_t rstd_nbytes, const float* gain, size_t gain_nbytes, void* grad_x,
                            size_t grad_x_nbytes, size_t grad_x_stride, float* grad_gain, size_t grad_gain_nbytes,
                            float* grad_bias, size_t grad_bias_nbytes, void* workspace, size_t workspace_nbytes,
                            size_t rows, size_t cols, int element);

/*
 * Of softmax(logits / temperature) for every row of `vocab` logits:
 *   log_prob       log probability of tokens[row]; 0 where the token is outside [0, vocab) (an ignored
 *                  position)
 *   entropy        -sum p log p
 *   lse            log sum exp(logits / temperature)
 *   top_ids, top_log_probs [rows, top]   the `top` likeliest tokens, 0 <= top <= MCC_MOST_TOP and <= vocab,
 *                  with their log probabilities: larger logit first, equal logits (-0 = +0) by the lower
 *                  token, NaN last
 * Every output may be null; tokens may be null (then log_prob is 0).  Logits of -inf (masked tokens) have
 * probability 0 and log probability -inf; in a row of -inf alone every log probability and lse are -inf
 * and the entropy is 0.  A NaN or +inf makes the row's outputs NaN but for top_ids.
 */
#define MCC_MOST_TOP 128
size_t mcc_token_log_probs_workspace_nbytes(size_t rows, size_t vocab, size_t top, int element);
int mcc_token_log_probs(void* stream, const void* logits, size_t logits_nbytes, size_t logits_stride,
                        const int32_t* tokens, size_t tokens_nbytes, float* log_prob, size_t log_prob_nbytes,
                        float* entropy, size_t entropy_nbytes, float* lse, size_t lse_nbytes, int32_t* top_ids,
                        size_t top_ids_nbytes, float* top_log_probs, size_t top_log_probs_nbytes, void* workspace,
                        size_t workspace_nbytes, size_t rows, size_t vocab, size_t top, int element, float temperature);

/*
 * Gradient of the logits for upstream gradients of log_prob and of entropy (either may be null), from the
 * forward call's lse and entropy (entropy is looked at only with grad_entropy):
 *   ((token == j) - p_j) * grad_log_prob - p_j (log p_j + entropy) * grad_entropy,  over temperature.
 * With grad_log_prob = -1 / n it is the gradient of the mean cross entropy.  Ignored positions take no
 * grad_log_prob.  Rows whose upstream gradients are zero and rows of -inf alone get zeros whatever their
 * logits hold.  p is taken as exp(logit / temperature - lse), so lse has to hold it: p's relative error grows
 * with |lse|, by 2^-24 |lse| (logits over the temperature in the thousands: 2^-12), and in a row whose
 * largest logit is so far from zero that its lse rounds log sum away (beyond 2^24, as the type's lowest
 * value used as a mask for the whole row) the gradient is not that of the uniform row; where lse leaves the
 * range of binary32 it is 0 (-inf) or NaN (+inf).  grad_logits may replace logits.
 */
int mcc_token_log_probs_backward(void* stream, const void* logits, size_t logits_nbytes, size_t logits_stride,
                                 const int32_t* tokens, size_t tokens_nbytes, const float* lse, size_t lse_nbytes,
                                 const float* entropy, size_t entropy_nbytes, const float* grad_log_prob,
                                 size_t grad_log_prob_nbytes, const float* grad_entropy, size_t grad_entropy_nbytes,
                                 void* grad_logits, size_t grad_logits_nbytes, size_t grad_logits_stride, size_t rows,
                                 size_t vocab, int element, float temperature);

/*
 * Distillation from a teacher's top logits, such as the top_ids and top_log_probs of
 * mcc_token_log_probs: with q = softmax(teacher_logits / temperature) over the row's entries and
 * p = softmax(logits / temperature) over the whole vocabulary,
 *   loss[row] = temperature^2 * sum q_i (log q_i - log p_id(i)),
 * and grad_logits = d(sum of weight[row] * loss[row]) / d logits = weight temperature (p_j - sum of the q_i with
 * id(i) = j).  teacher_ids and teacher_logits are [rows, top], 1 <= top <= MCC_MOST_TOP; an id outside
 * [0, vocab) is no entry (rows with fewer alternatives), an id may occur more than once.  weight (rows
 * floats; null: 1), loss and grad_logits may be null; loss is not weighted.  Rows without entries have
 * loss 0 and gradient 0, rows with weight 0 gradient 0 whatever their logits hold; a row of -inf alone has
 * loss +inf and gradient 0.  grad_logits may replace logits.
 */
int mcc_distill_top(void* stream, const void* logits, size_t logits_nbytes, size_t logits_stride,
                    const int32_t* teacher_ids, size_t teacher_ids_nbytes, const float* teacher_logits,
                    size_t teacher_logits_nbytes, const float* weight, size_t weight_nbytes, float* loss,
                    size_t loss_nbytes, void* grad_logits, size_t grad_logits_nbytes, size_t grad_logits_stride,
                    size_t rows, size_t vocab, size_t top, int element, float temperature);

/*
 * Device-resident storage.  Replaces the pooled VulkanRuntime::create_buffer /
 * Storage allocator (src/runtime/vulkan_backend.cpp:4663-4719,6462-6510;
 * src/tensor/storage.cpp:35-79): freed blocks are kept in power-of-two buckets
 * and reused; mcc_device_pool_clear returns them to the driver.  The byte
 * counters mirror device_bytes_current/peak (src/runtime/buffer.cpp:16-30).
 */
int mcc_device_alloc(void** ptr, size_t nbytes);
int mcc_device_free(void* ptr);
int mcc_device_pool_clear(void);
size_t mcc_device_bytes_current(void);
size_t mcc_device_bytes_peak(void);
void mcc_device_bytes_reset_peak(void);
int mcc_memcpy_h2d(void* stream, void* dst, const void* src, size_t nbytes);
int mcc_memcpy_d2h(void* stream, void* dst, const void* src, size_t nbytes);
int mcc_memset_zero(void* stream, void* dst, size_t nbytes);
/* Waits for everything enqueued on `stream` (Backend::finish,
 * src/runtime/backend.cpp:328-331). */
int mcc_stream_synchronize(void* stream);

/*
 * Per-kernel GPU timing.  While enabled, each kernel launched through this ABI is
 * bracketed by HIP events on its launch stream; mcc_profiler_query waits for them and
 * returns the summed duration and launch count of one kernel family:
 * "gemm_tn_f32", "counter_update", "counter_decode_weight", "counter_forward",
 * "counter_backward_input", "sgd_update", "adam_update", "layer_norm",
 * "layer_norm_backward", "token_log_probs", "token_log_probs_backward", "distill_top".  Replaces Profiler (src/runtime/profiler.cpp) and
 * VulkanRuntime::set_gpu_timing_enabled / last_gpu_time_us
 * (include/motifcl/runtime/vulkan_backend.hpp:181-185).
 */
void mcc_profiler_enable(int on);
void mcc_profiler_reset(void);
int mcc_profiler_query(const char* kernel_name, double* total_ms, uint64_t* launches);

#ifdef __cplusplus
}
#endif

#endif /* MOTIFCL_AMD_H */
