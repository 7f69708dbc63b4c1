// C ABI of the root-mean-square norm (include/rln.h, rln_rms_* and
// rln_dequantize): argument checks, launch shapes, the fixed-order reduction of
// the weight's gradient, and the widening of 8-bit values.

#include "rms_device.h"

namespace rln {
namespace rms {
namespace {

bool float_dtype(int dtype) {
    return dtype == RLN_DTYPE_F32 || dtype == RLN_DTYPE_F16 || dtype == RLN_DTYPE_BF16;
}

bool code_dtype(int dtype) {
    return dtype == RLN_DTYPE_INT8 || dtype == RLN_DTYPE_E4M3;
}

// Columns under one scale: 0 stands for the whole row.
bool valid_group(int64_t group) {
    return group == 0 || group == 32 || group == 64 || group == 128 || group == 256;
}

int64_t groups_of(int64_t hidden, int64_t group) {
    return group == 0 ? 1 : (hidden + group - 1) / group;
}

// log2 of a group's columns (valid ones are powers of two).
int group_shift(int64_t group) {
    int shift = 0;
    while (int64_t{1} << shift < group) {
        ++shift;
    }
    return shift;
}

int check_size(int64_t rows, int64_t hidden) {
    if (rows <= 0) {
        return fail(RLN_ERR_INVALID, "empty tensors are unsupported");
    }
    if (!rln_rms_hidden_supported(hidden)) {
        return fail(RLN_ERR_UNSUPPORTED, "unsupported RMSNorm hidden size: %lld",
                    static_cast<long long>(hidden));
    }
    if (rows > INT64_MAX / (hidden * 8)) {
        return fail(RLN_ERR_INVALID, "rows * hidden overflows int64");
    }
    return RLN_OK;
}

// A row stride in elements: any value whose last row's offset fits int64
// (0 for a row that is broadcast, negative ones walk backwards).
int check_stride(const char* name, int64_t stride, int64_t rows) {
    const int64_t limit = INT64_MAX / (8 * rows);
    if (stride > limit || stride < -limit) {
        return fail(RLN_ERR_INVALID, "%s: the row stride overflows int64", name);
    }
    return RLN_OK;
}

int64_t size_of(int dtype) {
    return dtype == RLN_DTYPE_F32 ? 4 : code_dtype(dtype) ? 1 : 2;
}

// Whether rows of `hidden` elements, `stride` elements apart from `pointer` on,
// start and end on whole 32-bit words: what Access::kWords asks.
bool whole_words(const void* pointer, int dtype, int64_t stride, int64_t hidden) {
    return reinterpret_cast<uintptr_t>(pointer) % 4 == 0 && stride * size_of(dtype) % 4 == 0
        && hidden * size_of(dtype) % 4 == 0;
}

int check_alignment(const char* name, const void* pointer, int dtype) {
    if (reinterpret_cast<uintptr_t>(pointer) % size_of(dtype) != 0) {
        return fail(RLN_ERR_INVALID, "%s is not aligned to its elements", name);
    }
    return RLN_OK;
}

// The checks the two forwards share, and the arguments they have in common.
int forward_args(const void* x, int x_dtype, int64_t x_stride, const void* branch,
                 int branch_dtype, int64_t branch_stride, const void* weight, int weight_dtype,
                 void* updated, void* output, int64_t rows, int64_t hidden, double eps,
                 void* stream, ForwardArgs* a) {
    int status = check_size(rows, hidden);
    if (status != RLN_OK) {
        return status;
    }
    if (!float_dtype(x_dtype)) {
        return fail(RLN_ERR_INVALID, "x must use float16, bfloat16 or float32");
    }
    if (branch != nullptr && !float_dtype(branch_dtype)) {
        return fail(RLN_ERR_INVALID, "branch must use float16, bfloat16 or float32");
    }
    if (!float_dtype(weight_dtype)) {
        return fail(RLN_ERR_INVALID, "weight must use float16, bfloat16 or float32");
    }
    if (!x || !weight || !output) {
        return fail(RLN_ERR_INVALID, "forward tensors must not be null");
    }
    if ((branch == nullptr) != (updated == nullptr)) {
        return fail(RLN_ERR_INVALID, "branch and updated must both be given or both be null");
    }
    if (!(eps >= 0.0)) {
        return fail(RLN_ERR_INVALID, "eps must not be negative");
    }
    if ((status = check_stride("x", x_stride, rows)) != RLN_OK
        || (status = check_stride("branch", branch_stride, rows)) != RLN_OK
        || (status = check_alignment("x", x, x_dtype)) != RLN_OK
        || (status = check_alignment("branch", branch, branch_dtype)) != RLN_OK
        || (status = check_alignment("weight", weight, weight_dtype)) != RLN_OK
        || (status = check_alignment("updated", updated, x_dtype)) != RLN_OK) {
        return status;
    }
    if ((status = check_stream(stream)) != RLN_OK) {
        return status;
    }
    *a = ForwardArgs{};
    a->x = x;
    a->branch = branch;
    a->weight = weight;
    a->updated = updated;
    a->normalized = output;
    a->x_stride = x_stride;
    a->branch_stride = branch_stride;
    a->rows = rows;
    a->hidden = static_cast<int>(hidden);
    a->weight_dtype = weight_dtype;
    a->eps = static_cast<float>(eps);
    a->inv_hidden = 1.0f / static_cast<float>(hidden);
    return RLN_OK;
}

int launch(ForwardArgs& a, int x_dtype, int branch_dtype, Mode mode, void* stream) {
    const Shape shape = forward_shape(a.rows, a.hidden, x_dtype);
    a.parts = shape.parts;
    a.row_lanes = shape.row_lanes;
    const int64_t hidden = a.hidden;
    a.words = whole_words(a.x, x_dtype, a.x_stride, hidden)
        && (a.branch == nullptr || whole_words(a.branch, branch_dtype, a.branch_stride, hidden))
        && whole_words(a.weight, a.weight_dtype, 0, hidden)
        && whole_words(a.updated, x_dtype, hidden, hidden)
        && whole_words(a.normalized, a.output_dtype, hidden, hidden)
        && (a.checkpoint == nullptr
            || whole_words(a.checkpoint, RLN_DTYPE_INT8, hidden, hidden));
    const hipStream_t queue = static_cast<hipStream_t>(stream);
    switch (x_dtype) {
        case RLN_DTYPE_F32:
            return launch_forward<float>(a, shape, branch_dtype, mode, queue);
        case RLN_DTYPE_F16:
            return launch_forward<half_t>(a, shape, branch_dtype, mode, queue);
        default:
            return launch_forward<bf16_t>(a, shape, branch_dtype, mode, queue);
    }
}

// Fixed-order sum of the partials [blocks][hidden] over the blocks, rounded
// once to the weight's type. A block owns 16 columns: 16 lanes read one 64-byte
// line of a partial row, its 64 groups of lanes take every 64th row each and
// add it in ascending order; the 64 sums are then added in ascending order.
// Narrow column blocks because the sum is latency-bound: at 4096 columns the
// 256 of them read the partials from every CU.
constexpr int kReduceColumns = 16;
constexpr int kReduceGroups = 64;

__global__ __launch_bounds__(kReduceColumns * kReduceGroups) void reduce_kernel(
    const float* __restrict__ partials, void* __restrict__ grad_weight, int dtype,
    int blocks, int hidden) {
    __shared__ float totals[kReduceGroups][kReduceColumns + 1];
    const int lane = threadIdx.x % kReduceColumns;
    const int group = threadIdx.x / kReduceColumns;
    const int column = blockIdx.x * kReduceColumns + lane;
    float total = 0.0f;
    if (column < hidden) {
#pragma unroll 4
        for (int block = group; block < blocks; block += kReduceGroups) {
            total += partials[static_cast<int64_t>(block) * hidden + column];
        }
    }
    totals[group][lane] = total;
    __syncthreads();
    if (group == 0 && column < hidden) {
        float sum = 0.0f;
#pragma unroll
        for (int other = 0; other < kReduceGroups; ++other) {
            sum += totals[other][lane];
        }
        store_one(grad_weight, dtype, column, sum);
    }
}

// values = codes * scale of their group: 8 codes per thread, vectors in row
// order (the last of a row may be short). A block takes a run of vectors; its
// first one's row and column come from one 64-bit division per block, the
// threads' from a 32-bit one.
struct DequantizeArgs {
    const int8_t* codes;
    const float* scale;
    void* values;
    int64_t vectors;      // rows * row_vectors
    int row_vectors;      // vectors per row
    int hidden;
    int group_shift;
    int groups;
    int code_dtype;
    int value_dtype;
};

constexpr int kDequantizeThreads = 256;

template <Access kAccess>
__global__ __launch_bounds__(kDequantizeThreads) void dequantize_kernel(DequantizeArgs a) {
    constexpr int N = 8;
    constexpr bool kRun = kAccess == Access::kWords;
    const int64_t step = static_cast<int64_t>(gridDim.x) * kDequantizeThreads;
    for (int64_t begin = static_cast<int64_t>(blockIdx.x) * kDequantizeThreads;
         begin < a.vectors; begin += step) {
        const int64_t begin_row = begin / a.row_vectors;
        const uint32_t from =
            static_cast<uint32_t>(begin - begin_row * a.row_vectors) + threadIdx.x;
        const uint32_t rows_on = from / static_cast<uint32_t>(a.row_vectors);
        const int column = static_cast<int>(from - rows_on * a.row_vectors) * N;
        const int64_t row = begin_row + rows_on;
        const bool live = begin + threadIdx.x < a.vectors;
        const float scale = live ? a.scale[row * a.groups + (column >> a.group_shift)] : 0.0f;
        // Whole vectors lie one after another over the rows, so the block's are
        // one run that starts at a uniform address; short ones go row by row.
        const int64_t left = a.vectors - begin;
        const int64_t first = kRun ? begin * N : row * a.hidden;
        const int place = kRun ? static_cast<int>(threadIdx.x) * N : column;
        const int extent = kRun
            ? static_cast<int>(left < kDequantizeThreads ? left : kDequantizeThreads) * N
            : live ? a.hidden : 0;
        auto raw = load<kAccess, int8_t, N>(a.codes + first, place, extent);
        settle<kAccess>(raw, place, extent);
        float values[N];
        if (a.code_dtype == RLN_DTYPE_E4M3) {
            widen_e4m3<N>(raw, values);
        } else {
            widen<int8_t, N>(raw, values);
        }
#pragma unroll
        for (int e = 0; e < N; ++e) {
            values[e] *= scale;
        }
        store_as<kAccess, kBackwardStores, N>(a.values, a.value_dtype, first, place, extent,
                                              values);
    }
}

}  // namespace
}  // namespace rms
}  // namespace rln

using namespace rln;
using namespace rln::rms;

extern "C" {

int rln_rms_hidden_supported(int64_t hidden) {
    return hidden >= 1 && hidden <= kMaxHidden ? 1 : 0;
}

int rln_rms_forward(
    const void* x, int x_dtype, int64_t x_stride,
    const void* branch, int branch_dtype, int64_t branch_stride,
    const void* weight, int weight_dtype,
    void* updated, void* normalized, int normalized_dtype, float* rstd,
    int8_t* checkpoint, float* checkpoint_scale,
    int64_t rows, int64_t hidden, double eps, void* stream) {
    clear_error();
    ForwardArgs a;
    int status = forward_args(x, x_dtype, x_stride, branch, branch_dtype, branch_stride, weight,
                              weight_dtype, updated, normalized, rows, hidden, eps, stream, &a);
    if (status != RLN_OK) {
        return status;
    }
    if (!float_dtype(normalized_dtype)) {
        return fail(RLN_ERR_INVALID, "normalized must use float16, bfloat16 or float32");
    }
    if ((status = check_alignment("normalized", normalized, normalized_dtype)) != RLN_OK) {
        return status;
    }
    if ((checkpoint == nullptr) != (checkpoint_scale == nullptr)) {
        return fail(RLN_ERR_INVALID,
                    "checkpoint and checkpoint_scale must both be given or both be null");
    }
    if ((status = check_alignment("rstd", rstd, RLN_DTYPE_F32)) != RLN_OK
        || (status = check_alignment("checkpoint_scale", checkpoint_scale, RLN_DTYPE_F32))
            != RLN_OK) {
        return status;
    }
    a.output_dtype = normalized_dtype;
    a.rstd = rstd;
    a.checkpoint = checkpoint;
    a.scale = checkpoint_scale;
    a.groups = static_cast<int>(groups_of(hidden, kCheckpointGroup));
    return launch(a, x_dtype, branch_dtype,
                  checkpoint != nullptr ? Mode::kCheckpoint : Mode::kNormalize, stream);
}

int rln_rms_quantize(
    const void* x, int x_dtype, int64_t x_stride,
    const void* branch, int branch_dtype, int64_t branch_stride,
    const void* weight, int weight_dtype,
    void* updated, void* quantized, int quantized_dtype, float* scale, int64_t group,
    int64_t rows, int64_t hidden, double eps, void* stream) {
    clear_error();
    ForwardArgs a;
    int status = forward_args(x, x_dtype, x_stride, branch, branch_dtype, branch_stride, weight,
                              weight_dtype, updated, quantized, rows, hidden, eps, stream, &a);
    if (status != RLN_OK) {
        return status;
    }
    if (!code_dtype(quantized_dtype)) {
        return fail(RLN_ERR_INVALID, "quantized must use int8 or float8_e4m3fn");
    }
    if (!valid_group(group)) {
        return fail(RLN_ERR_INVALID, "group must be 0 (the whole row), 32, 64, 128 or 256");
    }
    if (!scale) {
        return fail(RLN_ERR_INVALID, "forward tensors must not be null");
    }
    if ((status = check_alignment("scale", scale, RLN_DTYPE_F32)) != RLN_OK) {
        return status;
    }
    a.output_dtype = quantized_dtype;
    a.scale = scale;
    a.groups = static_cast<int>(groups_of(hidden, group));
    // One scale per row, also where a group is as long as the row.
    a.group_shift = a.groups == 1 ? kWholeRow : group_shift(group);
    return launch(a, x_dtype, branch_dtype, Mode::kQuantize, stream);
}

size_t rln_rms_backward_workspace_bytes(int64_t rows, int64_t hidden, int x_dtype) {
    if (rows <= 0 || !rln_rms_hidden_supported(hidden) || !float_dtype(x_dtype)
        || backward_slabs(rows, hidden)) {
        return 0;
    }
    return static_cast<size_t>(backward_blocks(rows, backward_shape(hidden, x_dtype)))
        * static_cast<size_t>(hidden) * sizeof(float);
}

int rln_rms_backward(
    const void* grad_updated, const void* grad_normalized, int grad_normalized_dtype,
    const void* updated, int64_t updated_stride, const int8_t* checkpoint,
    const float* checkpoint_scale, int x_dtype,
    const void* weight, int weight_dtype, const float* rstd,
    void* grad_x, void* grad_branch, int branch_dtype, void* grad_weight,
    int64_t rows, int64_t hidden, void* workspace, size_t workspace_bytes, void* stream) {
    clear_error();
    int status = check_size(rows, hidden);
    if (status != RLN_OK) {
        return status;
    }
    if (!float_dtype(x_dtype)) {
        return fail(RLN_ERR_INVALID, "x must use float16, bfloat16 or float32");
    }
    if (!float_dtype(grad_normalized_dtype)) {
        return fail(RLN_ERR_INVALID, "grad_normalized must use float16, bfloat16 or float32");
    }
    if (!float_dtype(weight_dtype)) {
        return fail(RLN_ERR_INVALID, "weight must use float16, bfloat16 or float32");
    }
    if (grad_branch != nullptr && !float_dtype(branch_dtype)) {
        return fail(RLN_ERR_INVALID, "branch must use float16, bfloat16 or float32");
    }
    if (!grad_normalized || !weight || !rstd || !grad_x) {
        return fail(RLN_ERR_INVALID, "backward tensors must not be null");
    }
    if ((updated == nullptr) == (checkpoint == nullptr)
        || (checkpoint == nullptr) != (checkpoint_scale == nullptr)) {
        return fail(RLN_ERR_INVALID,
                    "give either updated or checkpoint with checkpoint_scale");
    }
    if ((status = check_stride("updated", updated_stride, rows)) != RLN_OK
        || (status = check_alignment("grad_updated", grad_updated, x_dtype)) != RLN_OK
        || (status = check_alignment("grad_normalized", grad_normalized, grad_normalized_dtype))
            != RLN_OK
        || (status = check_alignment("updated", updated, x_dtype)) != RLN_OK
        || (status = check_alignment("weight", weight, weight_dtype)) != RLN_OK
        || (status = check_alignment("grad_x", grad_x, x_dtype)) != RLN_OK
        || (status = check_alignment("grad_branch", grad_branch, branch_dtype)) != RLN_OK
        || (status = check_alignment("grad_weight", grad_weight, weight_dtype)) != RLN_OK
        || (status = check_alignment("rstd", rstd, RLN_DTYPE_F32)) != RLN_OK
        || (status = check_alignment("checkpoint_scale", checkpoint_scale, RLN_DTYPE_F32))
            != RLN_OK
        || (status = check_alignment("workspace", workspace, RLN_DTYPE_F32)) != RLN_OK) {
        return status;
    }
    const Shape shape = backward_shape(hidden, x_dtype);
    const size_t needed = grad_weight != nullptr
        ? rln_rms_backward_workspace_bytes(rows, hidden, x_dtype) : 0;
    if (needed > 0 && (workspace == nullptr || workspace_bytes < needed)) {
        return fail(RLN_ERR_INVALID, "workspace too small: need %zu bytes, got %zu", needed,
                    workspace == nullptr ? static_cast<size_t>(0) : workspace_bytes);
    }
    if ((status = check_stream(stream)) != RLN_OK) {
        return status;
    }
    BackwardArgs a{};
    a.grad_updated = grad_updated;
    a.grad_normalized = grad_normalized;
    a.updated = updated;
    a.checkpoint = checkpoint;
    a.scale = checkpoint_scale;
    a.weight = weight;
    a.rstd = rstd;
    a.grad_x = grad_x;
    a.grad_branch = grad_branch;
    const bool slabs = grad_weight != nullptr && backward_slabs(rows, hidden);
    a.partials = grad_weight != nullptr && !slabs ? static_cast<float*>(workspace) : nullptr;
    a.grad_weight = grad_weight;
    const int slab_columns = kSlabLanes * columns_of(x_dtype);
    a.slabs = slabs ? static_cast<int>((hidden + slab_columns - 1) / slab_columns) : 0;
    a.updated_stride = updated_stride;
    a.rows = rows;
    a.hidden = static_cast<int>(hidden);
    a.parts = shape.parts;
    a.row_lanes = shape.row_lanes;
    a.groups = static_cast<int>(groups_of(hidden, kCheckpointGroup));
    a.weight_dtype = weight_dtype;
    a.branch_dtype = branch_dtype;
    a.inv_hidden = 1.0f / static_cast<float>(hidden);
    a.words = whole_words(grad_updated, x_dtype, hidden, hidden)
        && whole_words(grad_normalized, grad_normalized_dtype, hidden, hidden)
        && (updated == nullptr || whole_words(updated, x_dtype, updated_stride, hidden))
        && (checkpoint == nullptr || whole_words(checkpoint, RLN_DTYPE_INT8, hidden, hidden))
        && whole_words(weight, weight_dtype, 0, hidden)
        && whole_words(grad_x, x_dtype, hidden, hidden)
        && (grad_branch == nullptr || whole_words(grad_branch, branch_dtype, hidden, hidden));
    const hipStream_t queue = static_cast<hipStream_t>(stream);
    switch (x_dtype) {
        case RLN_DTYPE_F32:
            status = launch_backward<float>(a, shape, grad_normalized_dtype, queue);
            break;
        case RLN_DTYPE_F16:
            status = launch_backward<half_t>(a, shape, grad_normalized_dtype, queue);
            break;
        default:
            status = launch_backward<bf16_t>(a, shape, grad_normalized_dtype, queue);
            break;
    }
    if (status != RLN_OK || grad_weight == nullptr || slabs) {
        return status;
    }
    const unsigned blocks =
        static_cast<unsigned>((hidden + kReduceColumns - 1) / kReduceColumns);
    reduce_kernel<<<dim3(blocks), kReduceColumns * kReduceGroups, 0, queue>>>(
        a.partials, grad_weight, weight_dtype, static_cast<int>(backward_blocks(rows, shape)),
        a.hidden);
    return check_launch("rms reduce_kernel");
}

int rln_dequantize(
    const void* quantized, int quantized_dtype, const float* scale, int64_t group,
    void* values, int values_dtype, int64_t rows, int64_t hidden, void* stream) {
    clear_error();
    if (rows <= 0 || hidden <= 0) {
        return fail(RLN_ERR_INVALID, "empty tensors are unsupported");
    }
    if (hidden > INT32_MAX - 4096) {
        return fail(RLN_ERR_UNSUPPORTED, "unsupported row length: %lld",
                    static_cast<long long>(hidden));
    }
    if (rows > INT64_MAX / (hidden * 8)) {
        return fail(RLN_ERR_INVALID, "rows * hidden overflows int64");
    }
    if (!code_dtype(quantized_dtype)) {
        return fail(RLN_ERR_INVALID, "quantized must use int8 or float8_e4m3fn");
    }
    if (!float_dtype(values_dtype)) {
        return fail(RLN_ERR_INVALID, "values must use float16, bfloat16 or float32");
    }
    if (!valid_group(group)) {
        return fail(RLN_ERR_INVALID, "group must be 0 (the whole row), 32, 64, 128 or 256");
    }
    if (!quantized || !scale || !values) {
        return fail(RLN_ERR_INVALID, "dequantize tensors must not be null");
    }
    int status = RLN_OK;
    if ((status = check_alignment("scale", scale, RLN_DTYPE_F32)) != RLN_OK
        || (status = check_alignment("values", values, values_dtype)) != RLN_OK
        || (status = check_stream(stream)) != RLN_OK) {
        return status;
    }
    DequantizeArgs a{};
    a.codes = static_cast<const int8_t*>(quantized);
    a.scale = scale;
    a.values = values;
    a.row_vectors = static_cast<int>((hidden + 7) / 8);
    a.vectors = rows * a.row_vectors;
    a.hidden = static_cast<int>(hidden);
    a.groups = static_cast<int>(groups_of(hidden, group));
    a.group_shift = group == 0 ? kWholeRow : group_shift(group);
    a.code_dtype = quantized_dtype;
    a.value_dtype = values_dtype;
    int64_t blocks = (a.vectors + kDequantizeThreads - 1) / kDequantizeThreads;
    blocks = blocks < kMaxBlocks ? blocks : kMaxBlocks;
    const hipStream_t queue = static_cast<hipStream_t>(stream);
    if (hidden % 8 == 0 && whole_words(quantized, quantized_dtype, 0, 8)
        && whole_words(values, values_dtype, 0, 8)) {
        dequantize_kernel<Access::kWords>
            <<<dim3(static_cast<unsigned>(blocks)), kDequantizeThreads, 0, queue>>>(a);
    } else {
        dequantize_kernel<Access::kLanes>
            <<<dim3(static_cast<unsigned>(blocks)), kDequantizeThreads, 0, queue>>>(a);
    }
    return check_launch("rms dequantize_kernel");
}

}  // extern "C"
