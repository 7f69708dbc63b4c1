/*
 * rln.h - C ABI of the MI355X (gfx950) fused residual-add + dropout + LayerNorm
 * library, librln_gfx950.so.
 *
 * The operator, per row of `hidden` elements (H):
 *
 *   d = branch                                   (eval, or dropout_p == 0)
 *   d = round_to_branch_dtype(float(branch) * keep * 1/(1-p))   (training, p > 0)
 *   updated    = x + d                           (fp32)
 *   mean       = sum(updated) / H
 *   rstd       = 1 / sqrt(sum((updated - mean)^2) / H + eps)
 *   normalized = (updated - mean) * rstd * weight + bias
 *
 * and its first-order backward. This is the contract of the reference's
 * native entry points csrc/residual_layer_norm.h:10-42 and
 * csrc/residual_layer_norm_kernel.hip:425-545 (forward), :548-618 (input
 * gradients), :727-869 (weight/bias gradients).
 *
 * The same operator with a root-mean-square norm, its 8-bit output and its 8-bit
 * checkpoint are the rln_rms_* entry points and rln_dequantize below.
 *
 * Conventions shared by every entry point:
 *  - All pointers are device pointers on the calling thread's current HIP
 *    device, except `philox` (host pointer to a descriptor).
 *  - Tensors are dense row-major [rows, hidden] (rln_rms_*: where not given a
 *    stride); mean/rstd are [rows].
 *  - The dropout mask is `rows * hidden / 32` uint32 words: keep(r, c) is
 *    bit (c % 32) of word r * hidden / 32 + c / 32 - the reference's layout
 *    (csrc/residual_layer_norm_kernel.hip:500-511, :162-164).
 *  - `stream` is a hipStream_t (NULL = the legacy default stream) of the
 *    current device; a stream of another device is rejected with
 *    RLN_ERR_INVALID. Work is enqueued asynchronously; nothing synchronizes
 *    the host.
 *  - No entry point allocates device memory; rln_backward_noalloc also takes
 *    no workspace (it keeps a static per-device scratch instead).
 *  - Return value: RLN_OK, or an RLN_ERR_* code with a message available
 *    from rln_last_error() (thread-local, valid until the next call on the
 *    same thread).
 */
#ifndef RLN_H
#define RLN_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Element types of the branch, grad_branch, normalized and grad_normalized
 * tensors (x, updated, mean, rstd and the other gradients are always fp32). */
enum rln_dtype {
    RLN_DTYPE_F32 = 0,
    RLN_DTYPE_F16 = 1,
    RLN_DTYPE_BF16 = 2,
    /* 8-bit codes, of rln_rms_quantize and rln_dequantize only: */
    RLN_DTYPE_INT8 = 3, /* -127 .. 127 */
    RLN_DTYPE_E4M3 = 4  /* OCP float8 e4m3 (finite and NaN), +-448 */
};

enum rln_status {
    RLN_OK = 0,
    RLN_ERR_INVALID = 1,     /* bad argument: shape, range, null pointer */
    RLN_ERR_UNSUPPORTED = 2, /* valid request this build does not serve */
    RLN_ERR_HIP = 3          /* HIP runtime reported an error at launch */
};

/*
 * Philox4x32-10 stream selection for dropout. Mirrors torch's
 * at::PhiloxCudaState: outside graph capture the values are given directly;
 * under HIP graph capture the seed and base offset live in device memory and
 * are read when the kernel runs (effective offset = *offset_ptr + offset).
 * Replaces the seed/offset reservation at
 * csrc/residual_layer_norm_kernel.hip:1755-1780.
 *
 * `threads` selects the layout of the stream over the tensor:
 *  - 128, 192 or 256: the reference's own, the hipRAND Philox stream of its
 *    forward launched with that many threads per row (reference
 *    csrc/residual_layer_norm_kernel.hip:449-511; the reference's Python
 *    passes 128, or 192 for hidden 1024, gfx1010_kernels/_normalization_native.py:5-12).
 *    Same (seed, offset, threads) => the reference's mask, bit for bit.
 *    Hidden sizes 128, 256, 384, 512, 768 and 1024 only, and the offset
 *    (offset, plus *offset_ptr under capture) must be a multiple of 4, as
 *    torch's generator hands out.
 *  - 0: this library's layout, one Philox block per four consecutive columns
 *    (counter = (offset / 4, (row * hidden + column) / 4)); every hidden size.
 */
typedef struct rln_philox {
    uint64_t seed;             /* used when seed_ptr == NULL            */
    uint64_t offset;           /* absolute offset, or intra-graph delta */
    const int64_t* seed_ptr;   /* device pointer or NULL                */
    const int64_t* offset_ptr; /* device pointer or NULL                */
    int64_t threads;           /* 0, or 128 / 192 / 256 (see above)     */
} rln_philox_t;

/*
 * Forward. Replaces residual_layer_norm_forward_hip
 * (csrc/residual_layer_norm.h:10-24; csrc/residual_layer_norm_kernel.hip:1720-1827).
 *
 * x, updated: fp32 [rows, hidden]; branch: [rows, hidden] in `branch_dtype`;
 * normalized: [rows, hidden] in `normalized_dtype` (fp32 in the reference;
 * fp16/bf16 round the fp32 result to nearest even for a consumer that reads
 * half precision); weight, bias: fp32 [hidden]; mean, rstd: fp32 [rows].
 * dropout_mask: rln_mask_words(rows, hidden) uint32 words, written only when
 * training && dropout_p > 0 (may be NULL otherwise). `philox` is read only in
 * that case (may be NULL otherwise). The call consumes
 * rln_philox_increment(hidden, philox->threads) offset units of the Philox
 * stream.
 * zero_grad_weight, zero_grad_bias: both NULL, or fp32 [hidden] each, set to
 * zero by this launch: the weight/bias gradient sums of a later
 * rln_backward(..., accumulate_parameters = 1), which then needs no zeroing
 * launch of its own (the reference memsets them in its backward,
 * csrc/residual_layer_norm_kernel.hip:1895-1901; one launch fewer per
 * training step here).
 */
int rln_forward(
    const float* x,
    const void* branch,
    int branch_dtype,
    const float* weight,
    const float* bias,
    float* updated,
    void* normalized,
    int normalized_dtype,
    float* mean,
    float* rstd,
    uint32_t* dropout_mask,
    float* zero_grad_weight,
    float* zero_grad_bias,
    int64_t rows,
    int64_t hidden,
    double dropout_p,
    double eps,
    int training,
    const rln_philox_t* philox,
    void* stream);

/*
 * Backward. Replaces residual_layer_norm_backward_hip
 * (csrc/residual_layer_norm.h:27-42; csrc/residual_layer_norm_kernel.hip:1830-2036).
 *
 * grad_updated: fp32 [rows, hidden]; grad_normalized: [rows, hidden] in
 * `grad_normalized_dtype` (the dtype of the forward's normalized output);
 * either upstream gradient may be NULL, meaning zero (the reference
 * materializes zeros instead, csrc/residual_layer_norm_bindings.cpp:62-67).
 * grad_x: fp32 [rows, hidden]; grad_branch: [rows, hidden] in branch_dtype.
 * grad_weight, grad_bias: fp32 [hidden], both NULL to skip the parameter
 * gradients (they are skipped as well when grad_normalized is NULL; the
 * outputs are then left untouched).
 * deterministic != 0 selects the fixed-order two-stage reduction of the
 * parameter gradients (bitwise reproducible); 0 selects grouped fp32 atomics.
 * accumulate_parameters != 0 adds the parameter gradients to the values
 * already in grad_weight / grad_bias (gradient accumulation across calls, one
 * kernel launch in atomic mode); 0 overwrites them.
 * In atomic mode the launch adds partial sums into both arrays with fp32 atomics:
 * once per chunk of 32-64 rows and column throughout a single-step launch (most
 * launches below 4-16 million elements), once per block and column at the end of
 * a larger one.
 * Placement (speed only): measured at hidden = 768 on the larger kind (MI355X,
 * [8192, 768] with fp32 gradients): when grad_bias starts within 2 KiB of a
 * multiple of 32 KiB after grad_weight (and at some larger distances: 256 and 384
 * KiB, 4 MiB), both arrays fall on the same memory channels and those atomics take
 * about 3.7 times as long (6.2 instead of 1.7 us per backward); adjacent arrays
 * (two consecutive allocations of `hidden` floats, or one [2, hidden] buffer) are
 * fast. Single-step launches hardly depend on it ([1024, 384] 3.8 against 4.0 us;
 * [4096, 768], [2048, 1600] and [8192, 768] with 16-bit gradients not at all).
 * workspace: device scratch of at least
 * rln_backward_workspace_bytes(rows, hidden, deterministic) bytes, 16-byte
 * aligned (may be NULL when that size is 0).
 */
int rln_backward(
    const float* grad_updated,
    const void* grad_normalized,
    int grad_normalized_dtype,
    const float* updated,
    const float* weight,
    const float* mean,
    const float* rstd,
    const uint32_t* dropout_mask,
    float* grad_x,
    void* grad_branch,
    int branch_dtype,
    float* grad_weight,
    float* grad_bias,
    int64_t rows,
    int64_t hidden,
    double dropout_p,
    int training,
    int deterministic,
    int accumulate_parameters,
    void* workspace,
    size_t workspace_bytes,
    void* stream);

/* Scratch bytes rln_backward_noalloc keeps per device (see below). */
#define RLN_NOALLOC_SCRATCH_BYTES (4u << 20)

/*
 * Backward that allocates nothing and takes no workspace. It has
 * no counterpart in the reference: it is for callers that cannot allocate
 * device memory or pass a workspace (code under HIP graph capture, tight
 * serving loops, harnesses that forbid hipMalloc). Same arguments, checks and
 * results as rln_backward without workspace / workspace_bytes: the
 * deterministic weight/bias partials live in a library-owned static device
 * array of RLN_NOALLOC_SCRATCH_BYTES on each device (held until the process
 * ends; its address is looked up once per device on the first call). A call
 * whose partials need more (rln_backward_workspace_bytes(rows, hidden, 1)
 * above that, e.g. hidden above 2048 once the backward runs its full 256
 * blocks) fails with RLN_ERR_INVALID before any GPU work. Every call on a
 * device shares that device's scratch, and nothing in it needs clearing (each
 * call overwrites what it reads): calls that overlap on one device (different
 * streams, different host threads) race and must be ordered by the caller.
 * Atomic mode uses no scratch.
 */
int rln_backward_noalloc(
    const float* grad_updated,
    const void* grad_normalized,
    int grad_normalized_dtype,
    const float* updated,
    const float* weight,
    const float* mean,
    const float* rstd,
    const uint32_t* dropout_mask,
    float* grad_x,
    void* grad_branch,
    int branch_dtype,
    float* grad_weight,
    float* grad_bias,
    int64_t rows,
    int64_t hidden,
    double dropout_p,
    int training,
    int deterministic,
    int accumulate_parameters,
    void* stream);

/* Workspace bytes rln_backward needs (0 in atomic mode): the per-block
 * weight/bias partials of the deterministic reduction, which the reference
 * allocates itself (csrc/residual_layer_norm_kernel.hip:1870-1872). */
size_t rln_backward_workspace_bytes(
    int64_t rows,
    int64_t hidden,
    int deterministic);

/* Philox offset units one dropout forward consumes (torch's `increment`):
 * 4 for threads == 0; for the reference's layout its own
 * 4 * ceil(ceil(hidden / threads) / 4) (csrc/residual_layer_norm_kernel.hip:1766-1770).
 * 0 (with rln_last_error set) for an unsupported hidden / threads pair. */
uint64_t rln_philox_increment(int64_t hidden, int64_t threads);

/* Number of uint32 dropout-mask words for [rows, hidden] (the reference's
 * mask size, csrc/residual_layer_norm_kernel.hip:1750-1753, :162-164). */
int64_t rln_mask_words(int64_t rows, int64_t hidden);

/* 1 if the library serves rows of `hidden` values, else 0: the reference's
 * sizes 128, 256, 384, 512, 768 and 1024 (specialized kernels) and every
 * other multiple of 64 from 128 to 8192 (kernels with a run-time row length;
 * the reference compiles only the six, gfx1010_kernels/normalization.py:12). */
int rln_hidden_supported(int64_t hidden);

/* Writes up to `capacity` supported hidden sizes in ascending order; returns
 * how many exist (the reference's NATIVE_HIDDEN_SIZES,
 * gfx1010_kernels/normalization.py:12). */
int rln_supported_hidden_sizes(int64_t* out, int capacity);

/*
 * Root-mean-square norm with the residual's addition. It has no counterpart in
 * the reference, whose only norm is LayerNorm. Per row of `hidden` elements:
 *
 *   updated    = x + branch                       (added in fp32, rounded to x's type)
 *   rstd       = 1 / sqrt(sum(updated^2) / hidden + eps)
 *   normalized = updated * rstd * weight          (fp32, rounded to normalized's type)
 *
 * x, branch, weight and normalized each use fp32, fp16 or bf16; updated has x's
 * type. No output may overlap an input. x and branch are rows of consecutive
 * elements, `x_stride` and `branch_stride` elements apart (any value, 0 for one
 * row read by all);
 * updated and normalized are dense. Every address is aligned to its elements; more
 * is not asked. Any hidden from 1 to 16384 (rln_rms_hidden_supported).
 * branch and updated are both NULL for a norm without an addition (updated = x).
 * rstd: fp32 [rows] for the backward, or NULL.
 * checkpoint, checkpoint_scale: both NULL, or the 8-bit checkpoint of updated
 * for rln_rms_backward: int8 [rows, hidden] and fp32 [rows, ceil(hidden / 128)].
 * With m = max(|updated|, 2^-100) over a group of 128 columns (the last one
 * shorter), code = round(updated * (127 / m)) to nearest even and scale = m / 127,
 * each operation rounded once to fp32. A group that holds an infinity or a NaN
 * has NaN for its scale.
 */
int rln_rms_forward(
    const void* x,
    int x_dtype,
    int64_t x_stride,
    const void* branch,
    int branch_dtype,
    int64_t branch_stride,
    const void* weight,
    int weight_dtype,
    void* updated,
    void* normalized,
    int normalized_dtype,
    float* rstd,
    int8_t* checkpoint,
    float* checkpoint_scale,
    int64_t rows,
    int64_t hidden,
    double eps,
    void* stream);

/*
 * Backward of rln_rms_forward (no counterpart in the reference). Per row, with
 * u = updated, or checkpoint * checkpoint_scale where the checkpoint is given:
 *
 *   p = grad_normalized * weight
 *   g = grad_updated + rstd * (p - u * rstd * sum(p * u * rstd) / hidden)
 *   grad_x = g in x's type, grad_branch = g in the branch's type
 *   grad_weight = sum over the rows of grad_normalized * u * rstd, in the
 *                 weight's type, added in fp32 in a fixed order (bitwise
 *                 reproducible; the library's rln_backward offers both)
 *
 * grad_updated (x's type) may be NULL, meaning zero. Gradients are dense;
 * updated is rows `updated_stride` elements apart. grad_branch may be NULL
 * (no addition, or a branch of x's type, whose gradient is grad_x itself), and
 * so may grad_weight. No output may overlap an input (other blocks still read them
 * for grad_weight while grad_x is written). workspace: device scratch of
 * rln_rms_backward_workspace_bytes(rows, hidden, x_dtype) bytes, aligned to 4
 * (unused, may be NULL, without grad_weight or where that size is 0); nothing in
 * it needs clearing, and calls that overlap need one each.
 */
int rln_rms_backward(
    const void* grad_updated,
    const void* grad_normalized,
    int grad_normalized_dtype,
    const void* updated,
    int64_t updated_stride,
    const int8_t* checkpoint,
    const float* checkpoint_scale,
    int x_dtype,
    const void* weight,
    int weight_dtype,
    const float* rstd,
    void* grad_x,
    void* grad_branch,
    int branch_dtype,
    void* grad_weight,
    int64_t rows,
    int64_t hidden,
    void* workspace,
    size_t workspace_bytes,
    void* stream);

/* Workspace bytes rln_rms_backward needs for grad_weight: the per-block sums
 * of its fixed-order reduction (no counterpart in the reference); 0 for launches of at
 * most 1024 rows and 2^21 elements, which sum it in blocks of their own. */
size_t rln_rms_backward_workspace_bytes(
    int64_t rows,
    int64_t hidden,
    int x_dtype);

/*
 * rln_rms_forward with its output in 8 bits (no counterpart in the reference),
 * for a consumer that multiplies 8-bit activations. quantized: [rows, hidden] in
 * RLN_DTYPE_INT8 or RLN_DTYPE_E4M3; scale: fp32 [rows, groups], where `group` is the
 * number of columns under one scale, 32, 64, 128 or 256 (the last group of a
 * row may be shorter), or 0 for one scale per row. With v = updated * weight in
 * fp32, m = max(|v|, 2^-100) over the group and Q = 127 or 448:
 *
 *   code  = v * (Q / m), rounded to nearest even
 *   scale = (m / Q) * rstd;    normalized ~ code * scale
 *
 * each operation rounded once to fp32: rstd, a factor of the whole row, is in
 * the scale alone, so the codes do not depend on the order of any sum. A group
 * that holds an infinity or a NaN has NaN for its scale.
 */
int rln_rms_quantize(
    const void* x,
    int x_dtype,
    int64_t x_stride,
    const void* branch,
    int branch_dtype,
    int64_t branch_stride,
    const void* weight,
    int weight_dtype,
    void* updated,
    void* quantized,
    int quantized_dtype,
    float* scale,
    int64_t group,
    int64_t rows,
    int64_t hidden,
    double eps,
    void* stream);

/*
 * values = code * scale of the code's group, rounded to the values' type (fp32,
 * fp16 or bf16): what rln_rms_quantize wrote, for a consumer that does not read 8
 * bits (no counterpart in the reference). All tensors are dense; `group` as in
 * rln_rms_quantize, 1 <= hidden < 2^31 - 4096.
 */
int rln_dequantize(
    const void* quantized,
    int quantized_dtype,
    const float* scale,
    int64_t group,
    void* values,
    int values_dtype,
    int64_t rows,
    int64_t hidden,
    void* stream);

/* 1 if the rln_rms_* entry points serve rows of `hidden` values, 1 to 16384,
 * else 0 (no counterpart in the reference). */
int rln_rms_hidden_supported(int64_t hidden);

/*
 * Gated residual norm (rln_gated_*). It has no counterpart in the reference. Per
 * row of `hidden` elements, with gate and weight rows of as many:
 *
 *   a          = branch * branch_rstd * branch_weight,
 *                branch_rstd = 1 / sqrt(sum(branch^2) / hidden + branch_eps);
 *                a = branch where branch_weight is NULL
 *   updated    = residual_scale * x + branch_scale * gate * a
 *   rstd       = 1 / sqrt(sum(updated^2) / hidden + eps)     (of the rounded stream)
 *   normalized = updated * rstd * weight
 *
 * computed in fp32 and rounded once to the outputs' types. x, branch,
 * branch_weight, gate, weight and normalized each use fp32, fp16 or bf16; updated
 * has x's type.
 */

/* Rows of factors that repeat over the stream: row r of the stream takes row
 * r / rows of `data`, whose rows of consecutive elements are `stride` elements
 * apart. `rows` divides the number of the stream's rows: all of them for one row of
 * factors, 1 for one each. data is NULL for factors of one (of a gate). */
typedef struct rln_factor_t {
    const void* data;
    int dtype;
    int64_t stride;
    int64_t rows;
} rln_factor_t;

/*
 * Forward (no counterpart in the reference). x and branch are rows of consecutive
 * elements, `x_stride` and `branch_stride` elements apart (any value); branch_weight
 * is one row; updated and normalized are dense. No output may overlap an input.
 * Every address is aligned to its elements; more is not asked. gate may be NULL,
 * weight may not. Where gate and weight both repeat over some of the rows, they
 * repeat over the same. statistics: fp32 [2 * rows] for the backward (rstd, then
 * branch_rstd with a branch_weight), or NULL. Any hidden from 1 to 16384.
 */
int rln_gated_forward(
    const void* x,
    int x_dtype,
    int64_t x_stride,
    const void* branch,
    int branch_dtype,
    int64_t branch_stride,
    const void* branch_weight,
    int branch_weight_dtype,
    const rln_factor_t* gate,
    const rln_factor_t* weight,
    void* updated,
    void* normalized,
    int normalized_dtype,
    float* statistics,
    int64_t rows,
    int64_t hidden,
    double residual_scale,
    double branch_scale,
    double eps,
    double branch_eps,
    void* stream);

/*
 * Backward of rln_gated_forward (no counterpart in the reference). Per row, with
 * c = branch_scale * gate * branch_weight, v = updated * rstd, b = branch * branch_rstd:
 *
 *   p           = grad_normalized * weight
 *   g           = grad_updated + rstd * (p - v * sum(p * v) / hidden)
 *   grad_x      = residual_scale * g
 *   grad_branch = branch_rstd * (c * g - b * sum(c * g * b) / hidden), or c * g
 *                 without a branch_weight
 *   grad_gate   = branch_scale * branch_weight * g * b, grad_branch_weight =
 *                 branch_scale * gate * g * b, grad_weight = grad_normalized * v,
 *                 each summed in fp32 over the rows that share the factor, in a
 *                 fixed order (bitwise reproducible)
 *
 * grad_updated (x's type) and grad_normalized may be NULL, meaning zero. Gradients
 * are dense, in the types of what they belong to (grad_gate and grad_weight with a
 * row for each row of factors); updated is dense. grad_gate, grad_branch_weight and
 * grad_weight may each be NULL. No output may overlap an input. workspace: device
 * scratch of rln_gated_backward_workspace_bytes bytes, aligned to 4 (unused, may be
 * NULL, where none of the three is asked for, or grad_gate alone of a gate with a
 * row each); nothing in it needs clearing, and calls that overlap need one each.
 */
int rln_gated_backward(
    const void* grad_updated,
    const void* grad_normalized,
    int grad_normalized_dtype,
    const void* updated,
    int x_dtype,
    const void* branch,
    int branch_dtype,
    int64_t branch_stride,
    const void* branch_weight,
    int branch_weight_dtype,
    const rln_factor_t* gate,
    const rln_factor_t* weight,
    const float* statistics,
    void* grad_x,
    void* grad_branch,
    void* grad_gate,
    void* grad_branch_weight,
    void* grad_weight,
    int64_t rows,
    int64_t hidden,
    double residual_scale,
    double branch_scale,
    void* workspace,
    size_t workspace_bytes,
    void* stream);

/* Workspace bytes rln_gated_backward needs for its sums (no counterpart in the
 * reference). gate_rows and weight_rows are the factors' `rows`; without a gate,
 * gate_rows is `rows`. Every group of rows that shares its factors has sums of its
 * own, 8 bytes a column and more: a weight with a row each takes 8 bytes an element. */
size_t rln_gated_backward_workspace_bytes(
    int64_t rows,
    int64_t hidden,
    int x_dtype,
    int64_t gate_rows,
    int64_t weight_rows);

/*
 * Rotary positions of query and key heads, with the root-mean-square norm of each
 * head in front (rln_rotary_*; no counterpart in the reference). Per head h of
 * `size` elements of a token:
 *
 *   n = h * rstd * weight, rstd = 1 / sqrt(sum(h^2) / size + eps); n = h without a weight
 *   pair i of n turns by positions[axis i] * frequencies[i], an angle taken in fp64:
 *   (n1, n2) -> (n1 * cos - n2 * sin, n1 * sin + n2 * cos)
 *
 * where pair i is elements (i, i + pairs) of the head, or (2i, 2i + 1) with
 * `interleaved`; elements from 2 * pairs on are not turned. Computed in fp32,
 * rounded once to the heads' type (fp32, fp16 or bf16, that of all heads of a call).
 */

#define RLN_POSITIONS_I64 0
#define RLN_POSITIONS_I32 1
#define RLN_POSITIONS_F32 2

/* Heads [outer, inner, heads, size] with consecutive elements, strides in elements
 * (any values). data is NULL where there are none. */
typedef struct rln_heads_t {
    const void* data;
    int64_t outer_stride;
    int64_t token_stride;
    int64_t head_stride;
} rln_heads_t;

/* Positions [axes, outer, inner] by strides in elements, and the pairs they turn.
 * `axis_of_pair`: host memory, `pairs` values below `axes`, or NULL for axis 0. */
typedef struct rln_rotary_t {
    const void* positions;
    int positions_type;      /* RLN_POSITIONS_* */
    int64_t axis_stride;
    int64_t outer_stride;
    int64_t token_stride;
    const void* frequencies; /* fp32, or fp64 with wide_frequencies */
    int wide_frequencies;
    const uint8_t* axis_of_pair;
    int64_t axes;            /* 1 to 4 */
    int64_t pairs;           /* 2 * pairs <= size */
    int interleaved;
} rln_rotary_t;

/* One of the two tensors of heads of a call, q or k. */
typedef struct rln_rotary_side_t {
    rln_heads_t heads;       /* the forward's input */
    rln_heads_t grad;        /* backward: the gradient of its output */
    int64_t count;           /* heads per token; 0 for no such tensor */
    const void* weight;      /* [size], or NULL for heads without a norm */
    int weight_dtype;
    void* output;            /* dense: the turned heads, or the gradient of `heads` */
    void* grad_weight;       /* backward: [size] in the weight's type, or NULL */
} rln_rotary_side_t;

/*
 * Forward, of outer * inner tokens (no counterpart in the reference): q->output and
 * k->output from q->heads and k->heads. size is at most 256, outer * inner at most
 * 2^30 - 1, and each side has at most 65536 heads. No output may overlap an input.
 */
int rln_rotary_forward(
    const rln_rotary_side_t* q,
    const rln_rotary_side_t* k,
    int dtype,
    const rln_rotary_t* rotary,
    int64_t outer,
    int64_t inner,
    int64_t size,
    double eps,
    void* stream);

/*
 * Backward (no counterpart in the reference): q->output and k->output are the
 * gradients of q->heads and k->heads, from q->grad and k->grad and, with a norm, the
 * heads (heads.data is not read without one). With t the gradient turned back, n = h *
 * rstd and p = t * weight:
 *
 *   gradient = rstd * (p - n * sum(p * n) / size), or t without a norm
 *   grad_weight = t * n summed over tokens and heads in fp32, in a fixed order
 *
 * workspace: rln_rotary_backward_workspace_bytes of device scratch, aligned to 4
 * (unused, may be NULL, without a grad_weight); calls that overlap need one each.
 */
int rln_rotary_backward(
    const rln_rotary_side_t* q,
    const rln_rotary_side_t* k,
    int dtype,
    const rln_rotary_t* rotary,
    int64_t outer,
    int64_t inner,
    int64_t size,
    double eps,
    void* workspace,
    size_t workspace_bytes,
    void* stream);

/* Workspace bytes rln_rotary_backward needs for its sums (no counterpart in the
 * reference). */
size_t rln_rotary_backward_workspace_bytes(
    int64_t outer,
    int64_t inner,
    int64_t q_heads,
    int64_t k_heads,
    int64_t size,
    int64_t pairs,
    int dtype);

/* Thread-local message for the last failed call on this thread (the text of
 * the reference's TORCH_CHECK messages, csrc/residual_layer_norm_kernel.hip:26-166). */
const char* rln_last_error(void);

/* GPU architecture the device code was built for ("gfx950"; the reference
 * gates on "gfx1010", gfx1010_kernels/normalization.py:57). */
const char* rln_target_arch(void);

/* Library version string (the reference's package version is
 * gfx1010_kernels/__init__.py:22). */
const char* rln_version(void);

#ifdef __cplusplus
}
#endif

#endif /* RLN_H */
