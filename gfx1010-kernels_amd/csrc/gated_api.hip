// C ABI of the gated residual norm (include/rln.h, rln_gated_*): argument
// checks, launch shapes, and the fixed-order sums of its factors' gradients.

#include "gated_device.h"

namespace rln {
namespace gated {
namespace {

bool float_dtype(int dtype) {
    return dtype == RLN_DTYPE_F32 || dtype == RLN_DTYPE_F16 || dtype == RLN_DTYPE_BF16;
}

int64_t size_of(int dtype) {
    return dtype == RLN_DTYPE_F32 ? 4 : 2;
}

bool whole_words(const void* pointer, int dtype, int64_t stride, int64_t hidden) {
    return reinterpret_cast<uintptr_t>(pointer) % 4 == 0 && stride * size_of(dtype) % 4 == 0
        && hidden * size_of(dtype) % 4 == 0;
}

bool whole_words(const Factor& factor, int64_t hidden) {
    return whole_words(factor.data, factor.dtype, factor.stride, hidden);
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

// A tensor of rows: its type, its elements' alignment, and a stride whose last
// row's offset fits int64.
int check_rows(const char* name, const void* data, int dtype, int64_t stride, int64_t rows) {
    if (!float_dtype(dtype)) {
        return fail(RLN_ERR_INVALID, "%s must use float16, bfloat16 or float32", name);
    }
    if (reinterpret_cast<uintptr_t>(data) % size_of(dtype) != 0) {
        return fail(RLN_ERR_INVALID, "%s is not aligned to its elements", name);
    }
    const int64_t limit = INT64_MAX / (8 * rows);
    if (stride > limit || stride < -limit) {
        return fail(RLN_ERR_INVALID, "%s: the row stride overflows int64", name);
    }
    return RLN_OK;
}

int check_factor(const char* name, const rln_factor_t* given, int64_t rows, Factor* factor) {
    *factor = Factor{nullptr, 0, rows, RLN_DTYPE_F32, kShared, 0, 0};
    if (given == nullptr || given->data == nullptr) {
        return RLN_OK;
    }
    if (given->rows < 1 || rows % given->rows != 0) {
        return fail(RLN_ERR_INVALID, "%s: its rows must each serve a whole share of the rows",
                    name);
    }
    *factor = Factor{given->data, given->stride, given->rows, given->dtype, kShared, 0, 0};
    set_repeat(factor, rows);
    return check_rows(name, given->data, given->dtype, given->stride, rows / given->rows);
}

// Rows whose factors' gradients are summed together: those that share a row of
// gate and of weight. A gate with a row for each token has no such sum.
int group_rows(const Factor& gate, const Factor& weight, int64_t rows, int64_t* group) {
    const bool summed = gate.data != nullptr && gate.rows > 1 && gate.rows < rows;
    if (summed && weight.rows < rows && weight.rows != gate.rows) {
        return fail(RLN_ERR_UNSUPPORTED, "gate and weight must repeat over the same rows");
    }
    *group = summed ? gate.rows : weight.rows;
    return RLN_OK;
}

// What both passes are given alike.
int check_common(const void* branch, int branch_dtype, int64_t branch_stride,
                 const void* branch_weight, int branch_weight_dtype, const rln_factor_t* gate,
                 const rln_factor_t* weight, int x_dtype, int64_t rows, int64_t hidden,
                 double residual_scale, double branch_scale, Factor* gate_out,
                 Factor* weight_out, int64_t* group) {
    int status = check_size(rows, hidden);
    if (status != RLN_OK) {
        return status;
    }
    if (!float_dtype(x_dtype)) {
        return fail(RLN_ERR_INVALID, "x must use float16, bfloat16 or float32");
    }
    if (!branch || weight == nullptr || !weight->data) {
        return fail(RLN_ERR_INVALID, "branch and weight must not be null");
    }
    if (!__builtin_isfinite(residual_scale) || !__builtin_isfinite(branch_scale)) {
        return fail(RLN_ERR_INVALID, "residual_scale and branch_scale must be finite");
    }
    if ((status = check_rows("branch", branch, branch_dtype, branch_stride, rows)) != RLN_OK
        || (branch_weight != nullptr
            && (status = check_rows("branch_weight", branch_weight, branch_weight_dtype, 0, 1))
                != RLN_OK)
        || (status = check_factor("gate", gate, rows, gate_out)) != RLN_OK
        || (status = check_factor("weight", weight, rows, weight_out)) != RLN_OK) {
        return status;
    }
    return group_rows(*gate_out, *weight_out, rows, group);
}

// ----------------------------------------------------------------------------
// The sums of S and T over the units (gated_device.h), in a fixed order, and the
// factors' gradients from them. A block owns 32 columns, a 128-byte line of a unit's
// row, of one of the two sums (blockIdx.y). Its 32 slots of 32 lanes take `concurrent`
// groups at a time, 32 / concurrent slots each, which add every so manieth unit of
// their group in ascending order; the first slot of each group adds the others'
// totals, writes the group's gradients and keeps the sum over the groups it has
// seen, which are added last. Every thread's loads, and the additions' reads of LDS, are
// under way together: one after another they took 6.5 us at [8192, 768] and 16.7 at
// [4096, 8192], in blocks of 16 columns.

struct SumArgs {
    const float* partials;
    const void* branch_weight;
    Factor gate;
    void* grad_gate;  // of a gate that is summed; else null
    void* grad_branch_weight;
    void* grad_weight;
    int64_t groups;
    int64_t group_units;
    int concurrent;
    int hidden;
    int branch_weight_dtype;
    int weight_dtype;
    int gate_groups;    // each group has a gate of its own, or not
    int weight_groups;
    float branch_scale;
};

constexpr int kSumColumns = 32;
constexpr int kSumSlots = 32;

__device__ __forceinline__ float load_one(const void* tensor, int dtype, int64_t index) {
    if (dtype == RLN_DTYPE_F32) {
        return static_cast<const float*>(tensor)[index];
    }
    if (dtype == RLN_DTYPE_F16) {
        return static_cast<float>(static_cast<const half_t*>(tensor)[index]);
    }
    return static_cast<float>(static_cast<const bf16_t*>(tensor)[index]);
}

// The totals of slots slot, slot + step, ... below slot + count, in that order.
__device__ __forceinline__ float add_slots(const float (&totals)[kSumSlots][kSumColumns], int slot,
                                           int lane, int step, int count) {
    float values[kSumSlots];
#pragma unroll
    for (int i = 0; i < kSumSlots; ++i) {
        values[i] = i < count ? totals[slot + i * step][lane] : 0.0f;
    }
    float sum = values[0];
#pragma unroll
    for (int i = 1; i < kSumSlots; ++i) {
        sum += values[i];
    }
    return sum;
}

__global__ __launch_bounds__(kSumColumns * kSumSlots) void sum_units_kernel(SumArgs a) {
    __shared__ float totals[kSumSlots][kSumColumns];
    const bool first_sum = blockIdx.y == 0;  // S; else T
    if (first_sum ? a.grad_gate == nullptr && a.grad_branch_weight == nullptr
                  : a.grad_weight == nullptr) {
        return;
    }
    const int lane = threadIdx.x % kSumColumns;
    const int slot = threadIdx.x / kSumColumns;
    const int column = blockIdx.x * kSumColumns + lane;
    const bool live = column < a.hidden;
    const int slots = kSumSlots / a.concurrent;
    const int place = slot / slots;
    const int part = slot - place * slots;
    const float* partials = a.partials + (first_sum ? 0 : a.hidden) + column;
    const int64_t unit_stride = int64_t{2} * a.hidden;
    float over_groups = 0.0f;
    for (int64_t base = 0; base < a.groups; base += a.concurrent) {
        const int64_t group = base + place;
        const bool own = group < a.groups && live;
        float total = 0.0f;
        if (own) {
            const float* from = partials + (group * a.group_units + part) * unit_stride;
            const int64_t step = slots * unit_stride;
            constexpr int kBatch = 8;
            int64_t unit = part;
            for (; unit + (kBatch - 1) * slots < a.group_units; unit += kBatch * slots) {
                float values[kBatch];
#pragma unroll
                for (int i = 0; i < kBatch; ++i) {
                    values[i] = from[i * step];
                }
#pragma unroll
                for (int i = 0; i < kBatch; ++i) {
                    total += values[i];
                }
                from += kBatch * step;
            }
            for (; unit < a.group_units; unit += slots, from += step) {
                total += *from;
            }
        }
        totals[slot][lane] = total;
        __syncthreads();
        if (own && part == 0) {
            total = add_slots(totals, slot, lane, 1, slots);
            if (first_sum) {
                if (a.gate_groups) {
                    if (a.grad_gate != nullptr) {
                        const float post = a.branch_weight != nullptr
                            ? load_one(a.branch_weight, a.branch_weight_dtype, column) : 1.0f;
                        store_one(a.grad_gate, a.gate.dtype, group * a.hidden + column,
                                  a.branch_scale * post * total);
                    }
                    total *= load_one(a.gate.data, a.gate.dtype, group * a.gate.stride + column);
                }
            } else if (a.weight_groups) {
                store_one(a.grad_weight, a.weight_dtype, group * a.hidden + column, total);
            }
            over_groups += total;
        }
        __syncthreads();
    }
    totals[slot][lane] = over_groups;
    __syncthreads();
    if (slot == 0 && live) {
        over_groups = add_slots(totals, 0, lane, slots, a.concurrent);
        if (!first_sum) {
            if (!a.weight_groups) {
                store_one(a.grad_weight, a.weight_dtype, column, over_groups);
            }
            return;
        }
        // The gate of token gates is in S already.
        const bool shared_gate = a.gate.data != nullptr && a.gate.rows > 1 && !a.gate_groups;
        if (a.grad_gate != nullptr && shared_gate) {
            const float post = a.branch_weight != nullptr
                ? load_one(a.branch_weight, a.branch_weight_dtype, column) : 1.0f;
            store_one(a.grad_gate, a.gate.dtype, column, a.branch_scale * post * over_groups);
        }
        if (a.grad_branch_weight != nullptr) {
            const float gate = shared_gate ? load_one(a.gate.data, a.gate.dtype, column) : 1.0f;
            store_one(a.grad_branch_weight, a.branch_weight_dtype, column,
                      a.branch_scale * gate * over_groups);
        }
    }
}

}  // namespace
}  // namespace gated
}  // namespace rln

using namespace rln;
using namespace rln::gated;

extern "C" {

int rln_gated_forward(
    const void* x, int x_dtype, int64_t x_stride,
    const void* branch, int branch_dtype, int64_t branch_stride,
    const void* branch_weight, int branch_weight_dtype,
    const rln_factor_t* gate, const rln_factor_t* weight,
    void* updated, void* normalized, int normalized_dtype, float* statistics,
    int64_t rows, int64_t hidden, double residual_scale, double branch_scale,
    double eps, double branch_eps, void* stream) {
    clear_error();
    gated::ForwardArgs a{};
    int64_t group = 0;
    int status = check_common(branch, branch_dtype, branch_stride, branch_weight,
                              branch_weight_dtype, gate, weight, x_dtype, rows, hidden,
                              residual_scale, branch_scale, &a.gate, &a.weight, &group);
    if (status != RLN_OK) {
        return status;
    }
    if (!x || !updated || !normalized) {
        return fail(RLN_ERR_INVALID, "forward tensors must not be null");
    }
    if (!(eps >= 0.0) || !(branch_eps >= 0.0)) {
        return fail(RLN_ERR_INVALID, "eps must not be negative");
    }
    if ((status = check_rows("x", x, x_dtype, x_stride, rows)) != RLN_OK
        || (status = check_rows("updated", updated, x_dtype, 0, 1)) != RLN_OK
        || (status = check_rows("normalized", normalized, normalized_dtype, 0, 1)) != RLN_OK
        || (status = check_rows("statistics", statistics, RLN_DTYPE_F32, 0, 1)) != RLN_OK
        || (status = check_stream(stream)) != RLN_OK) {
        return status;
    }
    const Shape shape = pass_shape(rows, hidden, x_dtype, branch_weight != nullptr);
    a.x = x;
    a.branch = branch;
    a.branch_weight = branch_weight;
    a.updated = updated;
    a.normalized = normalized;
    a.statistics = statistics;
    a.x_stride = x_stride;
    a.branch_stride = branch_stride;
    a.rows = rows;
    a.hidden = static_cast<int>(hidden);
    a.split = split_of(shape);
    a.row_lanes = shape.row_lanes;
    a.branch_weight_dtype = branch_weight_dtype;
    a.output_dtype = normalized_dtype;
    a.residual_scale = static_cast<float>(residual_scale);
    a.branch_scale = static_cast<float>(branch_scale);
    a.eps = static_cast<float>(eps);
    a.branch_eps = static_cast<float>(branch_eps);
    a.inv_hidden = 1.0f / static_cast<float>(hidden);
    a.words = whole_words(x, x_dtype, x_stride, hidden)
        && whole_words(branch, branch_dtype, branch_stride, hidden)
        && (branch_weight == nullptr || whole_words(branch_weight, branch_weight_dtype, 0, hidden))
        && whole_words(a.gate, hidden) && whole_words(a.weight, hidden)
        && whole_words(updated, x_dtype, hidden, hidden)
        && whole_words(normalized, normalized_dtype, hidden, hidden);
    const hipStream_t queue = static_cast<hipStream_t>(stream);
    switch (x_dtype) {
        case RLN_DTYPE_F32:
            return gated::launch_forward<float>(a, shape, branch_dtype, queue);
        case RLN_DTYPE_F16:
            return gated::launch_forward<half_t>(a, shape, branch_dtype, queue);
        default:
            return gated::launch_forward<bf16_t>(a, shape, branch_dtype, queue);
    }
}

size_t rln_gated_backward_workspace_bytes(int64_t rows, int64_t hidden, int x_dtype,
                                          int64_t gate_rows, int64_t weight_rows) {
    if (rows <= 0 || !rln_rms_hidden_supported(hidden) || !float_dtype(x_dtype) || gate_rows < 1
        || weight_rows < 1 || rows % gate_rows != 0 || rows % weight_rows != 0) {
        return 0;
    }
    const int64_t group = gate_rows > 1 && gate_rows < rows ? gate_rows : weight_rows;
    const bool token_gate = gate_rows == 1 && rows > 1;
    return static_cast<size_t>(
               units_of(rows, group, token_gate, walk_shape(hidden, x_dtype)).count)
        * 2 * static_cast<size_t>(hidden) * sizeof(float);
}

int rln_gated_backward(
    const void* grad_updated, const void* grad_normalized, int grad_normalized_dtype,
    const void* updated, int x_dtype,
    const void* branch, int branch_dtype, int64_t branch_stride,
    const void* branch_weight, int branch_weight_dtype,
    const rln_factor_t* gate, const rln_factor_t* weight, const float* statistics,
    void* grad_x, void* grad_branch, void* grad_gate, void* grad_branch_weight,
    void* grad_weight, int64_t rows, int64_t hidden, double residual_scale,
    double branch_scale, void* workspace, size_t workspace_bytes, void* stream) {
    clear_error();
    gated::BackwardArgs a{};
    int status = check_common(branch, branch_dtype, branch_stride, branch_weight,
                              branch_weight_dtype, gate, weight, x_dtype, rows, hidden,
                              residual_scale, branch_scale, &a.gate, &a.weight, &a.group_rows);
    if (status != RLN_OK) {
        return status;
    }
    if (!updated || !statistics || !grad_x || !grad_branch) {
        return fail(RLN_ERR_INVALID, "backward tensors must not be null");
    }
    if (grad_gate != nullptr && a.gate.data == nullptr) {
        return fail(RLN_ERR_INVALID, "grad_gate without a gate");
    }
    if (grad_branch_weight != nullptr && branch_weight == nullptr) {
        return fail(RLN_ERR_INVALID, "grad_branch_weight without a branch_weight");
    }
    if ((grad_normalized != nullptr
         && (status = check_rows("grad_normalized", grad_normalized, grad_normalized_dtype, 0, 1))
             != RLN_OK)
        || (status = check_rows("grad_updated", grad_updated, x_dtype, 0, 1)) != RLN_OK
        || (status = check_rows("updated", updated, x_dtype, 0, 1)) != RLN_OK
        || (status = check_rows("statistics", statistics, RLN_DTYPE_F32, 0, 1)) != RLN_OK
        || (status = check_rows("grad_x", grad_x, x_dtype, 0, 1)) != RLN_OK
        || (status = check_rows("grad_branch", grad_branch, branch_dtype, 0, 1)) != RLN_OK
        || (status = check_rows("grad_gate", grad_gate, a.gate.dtype, 0, 1)) != RLN_OK
        || (branch_weight != nullptr
            && (status = check_rows("grad_branch_weight", grad_branch_weight, branch_weight_dtype,
                                    0, 1)) != RLN_OK)
        || (status = check_rows("grad_weight", grad_weight, a.weight.dtype, 0, 1)) != RLN_OK
        || (status = check_rows("workspace", workspace, RLN_DTYPE_F32, 0, 1)) != RLN_OK) {
        return status;
    }
    const bool token_gate = a.gate.data != nullptr && a.gate.rows == 1;
    const bool summed = grad_branch_weight != nullptr || grad_weight != nullptr
        || (grad_gate != nullptr && !token_gate);
    const size_t needed = summed
        ? rln_gated_backward_workspace_bytes(rows, hidden, x_dtype, a.gate.rows, a.weight.rows)
        : 0;
    if (needed > 0 && (workspace == nullptr || workspace_bytes < needed)) {
        return fail(RLN_ERR_INVALID, "workspace too small: need %zu bytes, got %zu", needed,
                    workspace == nullptr ? static_cast<size_t>(0) : workspace_bytes);
    }
    if ((status = check_stream(stream)) != RLN_OK) {
        return status;
    }
    const Shape shape = walk_shape(hidden, x_dtype);
    const Units units = units_of(rows, a.group_rows, token_gate && rows > 1, shape);
    a.grad_updated = grad_updated;
    a.grad_normalized = grad_normalized;
    a.updated = updated;
    a.branch = branch;
    a.branch_weight = branch_weight;
    a.statistics = statistics;
    a.grad_x = grad_x;
    a.grad_branch = grad_branch;
    a.grad_gate = token_gate ? grad_gate : nullptr;
    a.partials = summed ? static_cast<float*>(workspace) : nullptr;
    a.branch_stride = branch_stride;
    a.rows = rows;
    a.units = units.count;
    a.group_units = static_cast<int>(units.group_units);
    a.hidden = static_cast<int>(hidden);
    a.split = split_of(shape);
    a.row_lanes = shape.row_lanes;
    a.grad_dtype = grad_normalized_dtype;
    a.branch_weight_dtype = branch_weight_dtype;
    a.residual_scale = static_cast<float>(residual_scale);
    a.branch_scale = static_cast<float>(branch_scale);
    a.inv_hidden = 1.0f / static_cast<float>(hidden);
    a.words = whole_words(grad_updated, x_dtype, hidden, hidden)
        && (grad_normalized == nullptr
            || whole_words(grad_normalized, grad_normalized_dtype, hidden, hidden))
        && whole_words(updated, x_dtype, hidden, hidden)
        && whole_words(branch, branch_dtype, branch_stride, hidden)
        && (branch_weight == nullptr || whole_words(branch_weight, branch_weight_dtype, 0, hidden))
        && whole_words(a.gate, hidden) && whole_words(a.weight, hidden)
        && whole_words(grad_x, x_dtype, hidden, hidden)
        && whole_words(grad_branch, branch_dtype, hidden, hidden)
        && (a.grad_gate == nullptr || whole_words(a.grad_gate, a.gate.dtype, hidden, hidden));
    const hipStream_t queue = static_cast<hipStream_t>(stream);
    switch (x_dtype) {
        case RLN_DTYPE_F32:
            status = gated::launch_backward<float>(a, shape, branch_dtype, queue);
            break;
        case RLN_DTYPE_F16:
            status = gated::launch_backward<half_t>(a, shape, branch_dtype, queue);
            break;
        default:
            status = gated::launch_backward<bf16_t>(a, shape, branch_dtype, queue);
            break;
    }
    if (status != RLN_OK || !summed) {
        return status;
    }
    SumArgs sum{};
    sum.partials = a.partials;
    sum.branch_weight = branch_weight;
    sum.gate = a.gate;
    sum.grad_gate = token_gate ? nullptr : grad_gate;
    sum.grad_branch_weight = grad_branch_weight;
    sum.grad_weight = grad_weight;
    sum.groups = units.groups;
    sum.group_units = units.group_units;
    sum.concurrent = 1;
    while (sum.concurrent < units.groups && sum.concurrent < kSumSlots) {
        sum.concurrent *= 2;
    }
    sum.hidden = a.hidden;
    sum.branch_weight_dtype = branch_weight_dtype;
    sum.weight_dtype = a.weight.dtype;
    sum.gate_groups = !token_gate && a.gate.data != nullptr && a.gate.rows < rows;
    sum.weight_groups = a.weight.rows < rows;
    sum.branch_scale = a.branch_scale;
    const unsigned blocks = static_cast<unsigned>((hidden + kSumColumns - 1) / kSumColumns);
    sum_units_kernel<<<dim3(blocks, 2), kSumColumns * kSumSlots, 0, queue>>>(sum);
    return check_launch("gated sum_units_kernel");
}

}  // extern "C"
