// PyTorch glue for the root-mean-square norm's C ABI (include/rln.h, rln_rms_*
// and rln_dequantize); part of the module `gfx1010_kernels._C`:
//
//   residual_rms_norm(x, branch, weight, eps, normalized_dtype, checkpoint)
//       autograd op returning (updated, normalized); x itself as `updated`
//       without a branch
//   residual_rms_norm_if_supported(...)   the same, or None
//   residual_rms_norm_forward(...)        (updated, normalized, state)
//   residual_rms_norm_backward(...)       (grad_x, grad_branch, grad_weight)
//   residual_rms_norm_quantized(...)      (updated, quantized, scale)
//   dequantize(quantized, scale, group, dtype)
//   ..._if_supported(...)                 either of the two, or None
//
// The reference has no such operator. This file owns what the C ABI leaves to
// the caller: tensor allocation, row strides, the device guard and the current
// stream.

#include "rows_torch.h"

#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/dynamo/compiled_autograd.h>

#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>

#include <memory>
#include <mutex>
#include <optional>
#include <string>
#include <tuple>
#include <vector>

using namespace rln_glue;

namespace {

constexpr int64_t kCheckpointGroup = 128;

void check_inputs(const at::Tensor& x, const at::Tensor& branch, const at::Tensor& weight,
                  double eps) {
    TORCH_CHECK(x.is_cuda(), "x must be a HIP tensor");
    refuse_tangents("residual RMSNorm", {x, branch, weight});
    refuse_recording("residual RMSNorm");
    TORCH_CHECK((!branch.defined() || branch.is_cuda()) && weight.is_cuda(),
                "branch and weight must be HIP tensors");
    TORCH_CHECK(
        (!branch.defined() || branch.device() == x.device()) && weight.device() == x.device(),
        "all tensors must be on the same HIP device");
    TORCH_CHECK(supported_dtype(x.scalar_type()), "x must use float16, bfloat16 or float32");
    TORCH_CHECK(!branch.defined() || supported_dtype(branch.scalar_type()),
                "branch must use float16, bfloat16 or float32");
    TORCH_CHECK(supported_dtype(weight.scalar_type()),
                "weight must use float16, bfloat16 or float32");
    TORCH_CHECK(x.dim() >= 1, "x must have at least one dimension");
    TORCH_CHECK(!branch.defined() || branch.sizes() == x.sizes(), "branch must match x");
    const int64_t hidden = x.size(-1);
    TORCH_CHECK(rln_rms_hidden_supported(hidden), "unsupported RMSNorm hidden size: ", hidden);
    TORCH_CHECK(weight.sizes() == at::IntArrayRef({hidden}), "weight must match the hidden size");
    TORCH_CHECK(eps >= 0.0, "eps must not be negative");
}

// What a recorded forward keeps beside (or, with the checkpoint, in the place
// of) `updated`, in one allocation of bytes: rstd, the checkpoint's scales and
// its codes, each 256-byte aligned.
struct State {
    int64_t scale;
    int64_t codes;
    int64_t bytes;
};

State state_layout(int64_t rows, int64_t hidden, bool checkpoint) {
    const auto aligned = [](int64_t count) { return (count + 255) / 256 * 256; };
    const int64_t groups = (hidden + kCheckpointGroup - 1) / kCheckpointGroup;
    State state{};
    state.scale = aligned(4 * rows);
    state.codes = state.scale + (checkpoint ? aligned(4 * rows * groups) : 0);
    state.bytes = checkpoint ? state.codes + rows * hidden : 4 * rows;
    return state;
}

// updated is undefined without a branch; state, when given, receives what the
// backward needs. `rows_of_x` receives x as it was read (the input, or its copy).
std::tuple<at::Tensor, at::Tensor> forward_impl(
    const at::Tensor& x,
    const at::Tensor& branch,
    const at::Tensor& weight,
    double eps,
    std::optional<at::ScalarType> normalized_dtype,
    bool checkpoint,
    at::Tensor* state,
    at::Tensor* rows_of_x) {
    check_inputs(x, branch, weight, eps);
    const at::ScalarType output_type = normalized_dtype.value_or(x.scalar_type());
    TORCH_CHECK(supported_dtype(output_type),
                "normalized_dtype must be float32, float16 or bfloat16");
    c10::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
    const int64_t hidden = x.size(-1);
    const int64_t rows = x.numel() / hidden;
    auto updated = branch.defined() ? output_like(x, x.scalar_type()) : at::Tensor();
    auto normalized = output_like(x, output_type);
    State layout{};
    uint8_t* kept = nullptr;
    if (state != nullptr) {
        layout = state_layout(rows, hidden, checkpoint);
        *state = empty_device({layout.bytes}, at::kByte, x.device());
        kept = static_cast<uint8_t*>(state->data_ptr());
    }
    int64_t x_stride = 0;
    const auto x_rows = as_rows(x, &x_stride);
    if (rows_of_x != nullptr) {
        *rows_of_x = x_rows;
    }
    if (rows == 0) {
        return {updated, normalized};
    }
    int64_t branch_stride = 0;
    const auto branch_rows = branch.defined() ? as_rows(branch, &branch_stride) : branch;
    const auto weight_row = dense(weight);
    const bool codes = kept != nullptr && checkpoint;
    check_status(rln_rms_forward(
        x_rows.data_ptr(), dtype_of(x.scalar_type()), x_stride,
        branch.defined() ? branch_rows.data_ptr() : nullptr,
        branch.defined() ? dtype_of(branch.scalar_type()) : RLN_DTYPE_F32, branch_stride,
        weight_row.data_ptr(), dtype_of(weight.scalar_type()),
        branch.defined() ? updated.data_ptr() : nullptr, normalized.data_ptr(),
        dtype_of(output_type), reinterpret_cast<float*>(kept),
        codes ? reinterpret_cast<int8_t*>(kept + layout.codes) : nullptr,
        codes ? reinterpret_cast<float*>(kept + layout.scale) : nullptr,
        rows, hidden, eps, stream_of(x)));
    return {updated, normalized};
}

// grad_branch is undefined where it equals grad_x (no branch, or one of x's
// type), grad_weight where it is not asked for.
std::tuple<at::Tensor, at::Tensor, at::Tensor> backward_impl(
    const at::Tensor& grad_updated_in,
    const at::Tensor& grad_normalized_in,
    const at::Tensor& updated,
    const at::Tensor& state,
    const at::Tensor& weight,
    at::ScalarType x_type,
    std::optional<at::ScalarType> branch_type,
    bool checkpoint,
    bool weight_gradient) {
    TORCH_CHECK(grad_normalized_in.is_cuda(), "grad_normalized must be a HIP tensor");
    refuse_tangents("residual RMSNorm", {grad_updated_in, grad_normalized_in, updated, weight});
    refuse_recording("residual RMSNorm's backward");
    const auto device = grad_normalized_in.device();
    TORCH_CHECK(
        (!grad_updated_in.defined() || grad_updated_in.device() == device)
            && state.device() == device && weight.device() == device
            && (checkpoint || updated.device() == device),
        "all backward tensors must be on the same HIP device");
    TORCH_CHECK(supported_dtype(x_type) && (!branch_type || supported_dtype(*branch_type))
                    && supported_dtype(weight.scalar_type()),
                "x, branch and weight must use float16, bfloat16 or float32");
    TORCH_CHECK(supported_dtype(grad_normalized_in.scalar_type()),
                "grad_normalized must use float32, float16 or bfloat16");
    TORCH_CHECK(grad_normalized_in.dim() >= 1, "grad_normalized must have a dimension");
    TORCH_CHECK(
        !grad_updated_in.defined()
            || (grad_updated_in.scalar_type() == x_type
                && grad_updated_in.sizes() == grad_normalized_in.sizes()),
        "grad_updated must match grad_normalized's shape and x's type");
    const int64_t hidden = grad_normalized_in.size(-1);
    TORCH_CHECK(rln_rms_hidden_supported(hidden), "unsupported RMSNorm hidden size: ", hidden);
    TORCH_CHECK(weight.sizes() == at::IntArrayRef({hidden}), "weight must match the hidden size");
    const int64_t rows = grad_normalized_in.numel() / hidden;
    const State layout = state_layout(rows, hidden, checkpoint);
    TORCH_CHECK(state.scalar_type() == at::kByte && state.is_contiguous()
                    && state.numel() == layout.bytes,
                "state is not the forward's");
    int64_t updated_stride = 0;
    at::Tensor updated_rows;
    if (!checkpoint) {
        TORCH_CHECK(updated.scalar_type() == x_type
                        && updated.sizes() == grad_normalized_in.sizes(),
                    "updated must match grad_normalized's shape and x's type");
        updated_rows = as_rows(updated, &updated_stride);
    }
    c10::hip::HIPGuardMasqueradingAsCUDA guard(device);
    const auto grad_normalized = dense(grad_normalized_in);
    const auto grad_updated = dense(grad_updated_in);
    const auto weight_row = dense(weight);
    auto grad_x = empty_device(grad_normalized.sizes(), x_type, device);
    auto grad_branch = branch_type && *branch_type != x_type
        ? empty_device(grad_normalized.sizes(), *branch_type, device) : at::Tensor();
    at::Tensor grad_weight;
    at::Tensor workspace;
    size_t bytes = 0;
    if (weight_gradient) {
        if (rows == 0) {
            grad_weight = at::zeros({hidden}, weight.options());
        } else {
            grad_weight = empty_device({hidden}, weight.scalar_type(), device);
            bytes = rln_rms_backward_workspace_bytes(rows, hidden, dtype_of(x_type));
            if (bytes > 0) {
                workspace = empty_device({static_cast<int64_t>(bytes)}, at::kByte, device);
            }
        }
    }
    if (rows == 0) {
        return {grad_x, grad_branch, grad_weight};
    }
    uint8_t* kept = static_cast<uint8_t*>(state.data_ptr());
    check_status(rln_rms_backward(
        grad_updated.defined() ? grad_updated.data_ptr() : nullptr, grad_normalized.data_ptr(),
        dtype_of(grad_normalized.scalar_type()),
        checkpoint ? nullptr : updated_rows.data_ptr(), updated_stride,
        checkpoint ? reinterpret_cast<const int8_t*>(kept + layout.codes) : nullptr,
        checkpoint ? reinterpret_cast<const float*>(kept + layout.scale) : nullptr,
        dtype_of(x_type), weight_row.data_ptr(), dtype_of(weight.scalar_type()),
        reinterpret_cast<const float*>(kept), grad_x.data_ptr(),
        grad_branch.defined() ? grad_branch.data_ptr() : nullptr,
        branch_type ? dtype_of(*branch_type) : RLN_DTYPE_F32,
        weight_gradient ? grad_weight.data_ptr() : nullptr, rows, hidden,
        workspace.defined() ? workspace.data_ptr() : nullptr, bytes, stream_of(grad_x)));
    return {grad_x, grad_branch, grad_weight};
}

// The graph's node, with edges to x, branch (none without one) and weight. A node
// of its own instead of a torch::autograd::Function: no map of saved values to
// fill and search in every call. Measured with empty bodies and three inputs, a
// forward costs 1.4 instead of 4.0 us and a backward 1 us less on the host, which
// small training steps are bound by.
class ResidualRmsNormBackward : public torch::autograd::Node {
 public:
    // updated (x without a branch), or undefined with the checkpoint.
    torch::autograd::SavedVariable kept;
    torch::autograd::SavedVariable weight;
    torch::autograd::SavedVariable state;
    at::ScalarType x_type = at::kFloat;
    std::optional<at::ScalarType> branch_type;
    bool checkpoint = false;

    std::string name() const override {
        return "ResidualRmsNormBackward";
    }

    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        kept.reset_data();
        weight.reset_data();
        state.reset_data();
    }

    // Gradients of (updated, normalized), or of normalized without a branch;
    // either may be undefined.
    torch::autograd::variable_list apply(torch::autograd::variable_list&& grads) override {
        std::lock_guard<std::mutex> lock(mutex_);
        if (!grads[branch_type ? 1 : 0].defined()) {
            Held held;  // the addition's gradient needs nothing that is kept
            held.branch_type = branch_type;
            return gradients(grads, held);
        }
        return gradients(grads, unpack());
    }

    // Compiled autograd: what the node holds, and its gradients as one call that the
    // compiled graph makes with its own tensors.
    void compiled_args(torch::dynamo::autograd::CompiledNodeArgs& args) const override {
        if (!checkpoint) {
            args.collect(kept, branch_type.has_value());
        }
        args.collect(weight, false);
        args.collect(state, false);
        args.collect(x_type);
        args.collect(branch_type);
        args.collect(checkpoint);
    }

    torch::autograd::variable_list apply_with_saved(
        const torch::autograd::variable_list& grads,
        torch::dynamo::autograd::SwapSavedVariables& saved) override {
        namespace compiled = torch::dynamo::autograd;
        if (!checkpoint) {
            saved.before(kept);
        }
        saved.before(weight);
        saved.before(state);
        const Held held = unpack();
        compiled::PackedArgs packed;
        packed.pack(held.kept.defined() ? std::optional(held.kept) : std::nullopt);
        packed.pack(held.weight);
        packed.pack(held.state);
        packed.pack(held.x_type);
        packed.pack(held.branch_type);
        packed.pack(held.checkpoint);
        packed.pack(held.weight_gradient);
        const auto call = [](const torch::autograd::variable_list& grads,
                             const std::vector<c10::IValue>& args) {
            compiled::PackedArgs given(args);
            Held held;
            held.kept = given.unpack<std::optional<at::Tensor>>().value_or(at::Tensor());
            held.weight = given.unpack<at::Tensor>();
            held.state = given.unpack<at::Tensor>();
            held.x_type = given.unpack<at::ScalarType>();
            held.branch_type = given.unpack<std::optional<at::ScalarType>>();
            held.checkpoint = given.unpack<bool>();
            held.weight_gradient = given.unpack<bool>();
            return gradients(grads, held);
        };
        const auto& compiler = compiled::getPyCompilerInterface();
        const std::string function = compiler->bind_function(
            saved.get_py_compiler(), name(), call,
            {compiled::IValuePacker<std::optional<at::Tensor>>::packed_type(),
             compiled::IValuePacker<at::Tensor>::packed_type(),
             compiled::IValuePacker<at::Tensor>::packed_type(),
             compiled::IValuePacker<at::ScalarType>::packed_type(),
             compiled::IValuePacker<std::optional<at::ScalarType>>::packed_type(),
             compiled::IValuePacker<bool>::packed_type(),
             compiled::IValuePacker<bool>::packed_type()},
            /*is_custom_function=*/true, /*is_traceable=*/false);
        auto results = compiler->call_function(
            saved.get_py_compiler(), "apply_functional", function, grads, packed.vec(),
            compiled::IValuePacker<std::vector<std::optional<torch::autograd::InputMetadata>>>::
                pack(compiled::get_input_metadata(next_edges())));
        if (!checkpoint) {
            saved.after(kept);
        }
        saved.after(weight);
        saved.after(state);
        return results;
    }

 private:
    // What the gradients are computed from.
    struct Held {
        at::Tensor kept;
        at::Tensor weight;
        at::Tensor state;
        at::ScalarType x_type = at::kFloat;
        std::optional<at::ScalarType> branch_type;
        bool checkpoint = false;
        bool weight_gradient = false;
    };

    Held unpack() {
        return Held{checkpoint ? at::Tensor() : kept.unpack(branch_type ? getptr() : nullptr),
                    weight.unpack(), state.unpack(), x_type, branch_type, checkpoint,
                    task_should_compute_output(2)};
    }

    static torch::autograd::variable_list gradients(const torch::autograd::variable_list& grads,
                                                    const Held& held) {
        const at::Tensor grad_updated = held.branch_type ? grads[0] : at::Tensor();
        const at::Tensor grad_normalized = held.branch_type ? grads[1] : grads[0];
        at::Tensor grad_x;
        at::Tensor grad_branch;
        at::Tensor grad_weight;
        if (grad_normalized.defined()) {
            std::tie(grad_x, grad_branch, grad_weight) = backward_impl(
                grad_updated, grad_normalized, held.kept, held.state, held.weight, held.x_type,
                held.branch_type, held.checkpoint, held.weight_gradient);
            if (held.branch_type && !grad_branch.defined()) {
                grad_branch = grad_x;  // one tensor, as for any addition
            }
            if (at::GradMode::is_enabled()) {
                // create_graph: the gradients are constants of a backward that
                // has none of its own; differentiating them again raises.
                refuse_second_order(
                    {grad_updated, grad_normalized, held.kept, held.weight},
                    {grad_x, grad_branch.is_same(grad_x) ? at::Tensor() : grad_branch,
                     grad_weight});
            }
        } else if (grad_updated.defined()) {
            grad_x = grad_updated;
            grad_branch = grad_updated.to(*held.branch_type);
        }
        return {grad_x, grad_branch, grad_weight};
    }

    static void refuse_second_order(const torch::autograd::variable_list& inputs,
                                    const torch::autograd::variable_list& outputs) {
        if (!torch::autograd::any_variable_requires_grad(inputs)) {
            return;
        }
        torch::autograd::variable_list given;
        for (const auto& input : inputs) {
            if (input.defined()) {
                given.push_back(input);
            }
        }
        const auto refusal = std::make_shared<torch::autograd::NotImplemented>(
            "residual_rms_norm (second-order gradients)",
            torch::autograd::collect_next_edges(given));
        for (const auto& output : outputs) {
            if (output.defined()) {
                torch::autograd::set_history(output, refusal);
            }
        }
    }
};

// Whether a call on these inputs has a gradient to record.
bool recorded(const at::Tensor& x, const at::Tensor& branch, const at::Tensor& weight) {
    return at::GradMode::is_enabled()
        && (x.requires_grad() || (branch.defined() && branch.requires_grad())
            || weight.requires_grad());
}

// (updated, normalized); x itself is `updated` without a branch.
std::tuple<at::Tensor, at::Tensor> residual_rms_norm(
    const at::Tensor& x,
    const std::optional<at::Tensor>& branch_in,
    const at::Tensor& weight,
    double eps,
    std::optional<at::ScalarType> normalized_dtype,
    bool checkpoint) {
    const at::Tensor branch = branch_in.value_or(at::Tensor());
    if (!recorded(x, branch, weight)) {
        // Nothing to record: no state is kept, and no checkpoint written.
        auto [updated, normalized] =
            forward_impl(x, branch, weight, eps, normalized_dtype, false, nullptr, nullptr);
        return {branch.defined() ? updated : x, normalized};
    }
    at::Tensor state;
    at::Tensor rows_of_x;
    at::Tensor updated;
    at::Tensor normalized;
    {
        // The kernels' own outputs; nothing inside records a graph.
        at::AutoDispatchBelowADInplaceOrView below;
        std::tie(updated, normalized) = forward_impl(
            x, branch, weight, eps, normalized_dtype, checkpoint, &state, &rows_of_x);
    }
    auto node = std::shared_ptr<ResidualRmsNormBackward>(new ResidualRmsNormBackward(),
                                                         torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(x, branch, weight));
    node->x_type = x.scalar_type();
    node->checkpoint = checkpoint;
    if (branch.defined()) {
        node->branch_type = branch.scalar_type();
        torch::autograd::set_history(updated, node);
    }
    torch::autograd::set_history(normalized, node);
    if (!checkpoint) {
        // An output is saved as one (no cycle through its own node); an input,
        // or the copy of its rows, as an input.
        node->kept = branch.defined()
            ? torch::autograd::SavedVariable(updated, true)
            : torch::autograd::SavedVariable(row_stride(x) ? x : rows_of_x, false);
    }
    node->weight = torch::autograd::SavedVariable(weight, false);
    node->state = torch::autograd::SavedVariable(state, false);
    return {branch.defined() ? updated : x, normalized};
}

// Whether the native path serves these inputs: what check_inputs asks, as one
// bool (the reason is worked out in Python when this is false).
bool rms_inputs_supported(const at::Tensor& x, const at::Tensor& branch,
                          const at::Tensor& weight, double eps) {
    if (!x.is_cuda() || x.dim() < 1 || !supported_dtype(x.scalar_type())
        || !weight.is_cuda() || weight.device() != x.device()
        || !supported_dtype(weight.scalar_type())) {
        return false;
    }
    if (branch.defined()
        && (!branch.is_cuda() || branch.device() != x.device() || branch.sizes() != x.sizes()
            || !supported_dtype(branch.scalar_type()))) {
        return false;
    }
    if (has_tangent(x) || has_tangent(branch) || has_tangent(weight)) {
        return false;
    }
    const int64_t hidden = x.size(-1);
    return rln_rms_hidden_supported(hidden) && weight.sizes() == at::IntArrayRef({hidden})
        && eps >= 0.0;
}

std::optional<std::tuple<at::Tensor, at::Tensor>> residual_rms_norm_if_supported(
    const at::Tensor& x,
    const std::optional<at::Tensor>& branch,
    const at::Tensor& weight,
    double eps,
    std::optional<at::ScalarType> normalized_dtype,
    bool checkpoint) {
    if (graph_recorded()
        || !rms_inputs_supported(x, branch.value_or(at::Tensor()), weight, eps)) {
        return std::nullopt;
    }
    return residual_rms_norm(x, branch, weight, eps, normalized_dtype, checkpoint);
}

// The pieces of the autograd op, for the registered custom ops. `updated` is an
// empty tensor without a branch.
std::tuple<at::Tensor, at::Tensor, at::Tensor> residual_rms_norm_forward(
    const at::Tensor& x,
    const std::optional<at::Tensor>& branch_in,
    const at::Tensor& weight,
    double eps,
    std::optional<at::ScalarType> normalized_dtype,
    bool checkpoint) {
    const at::Tensor branch = branch_in.value_or(at::Tensor());
    at::Tensor state;
    auto [updated, normalized] =
        forward_impl(x, branch, weight, eps, normalized_dtype, checkpoint, &state, nullptr);
    return {branch.defined() ? updated : empty_device({0}, x.scalar_type(), x.device()),
            normalized, state};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> residual_rms_norm_backward(
    const std::optional<at::Tensor>& grad_updated,
    const at::Tensor& grad_normalized,
    const std::optional<at::Tensor>& updated,
    const at::Tensor& state,
    const at::Tensor& weight,
    at::ScalarType x_type,
    std::optional<at::ScalarType> branch_type,
    bool checkpoint,
    bool weight_gradient) {
    TORCH_CHECK(checkpoint || (updated.has_value() && updated->defined()),
                "updated must be given without the checkpoint");
    return backward_impl(grad_updated.value_or(at::Tensor()), grad_normalized,
                         updated.value_or(at::Tensor()), state, weight, x_type, branch_type,
                         checkpoint, weight_gradient);
}

bool code_type(at::ScalarType type) {
    return type == at::kChar || type == at::kFloat8_e4m3fn;
}

int code_of(at::ScalarType type) {
    return type == at::kChar ? RLN_DTYPE_INT8 : RLN_DTYPE_E4M3;
}

std::vector<int64_t> scale_sizes(at::IntArrayRef sizes, int64_t group) {
    std::vector<int64_t> out(sizes.begin(), sizes.end());
    out.back() = group == 0 ? 1 : (out.back() + group - 1) / group;
    return out;
}

void check_group(int64_t group) {
    TORCH_CHECK(group == 0 || group == 32 || group == 64 || group == 128 || group == 256,
                "group_size must be None, 32, 64, 128 or 256");
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> residual_rms_norm_quantized(
    const at::Tensor& x,
    const std::optional<at::Tensor>& branch_in,
    const at::Tensor& weight,
    double eps,
    at::ScalarType dtype,
    int64_t group) {
    const at::Tensor branch = branch_in.value_or(at::Tensor());
    check_inputs(x, branch, weight, eps);
    TORCH_CHECK(code_type(dtype), "dtype must be int8 or float8_e4m3fn");
    check_group(group);
    c10::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
    const int64_t hidden = x.size(-1);
    const int64_t rows = x.numel() / hidden;
    auto updated = branch.defined() ? output_like(x, x.scalar_type()) : x;
    auto quantized = output_like(x, dtype);
    auto scale = empty_device(scale_sizes(x.sizes(), group), at::kFloat, x.device());
    if (rows == 0) {
        return {updated, quantized, scale};
    }
    int64_t x_stride = 0;
    const auto x_rows = as_rows(x, &x_stride);
    int64_t branch_stride = 0;
    const auto branch_rows = branch.defined() ? as_rows(branch, &branch_stride) : branch;
    const auto weight_row = dense(weight);
    check_status(rln_rms_quantize(
        x_rows.data_ptr(), dtype_of(x.scalar_type()), x_stride,
        branch.defined() ? branch_rows.data_ptr() : nullptr,
        branch.defined() ? dtype_of(branch.scalar_type()) : RLN_DTYPE_F32, branch_stride,
        weight_row.data_ptr(), dtype_of(weight.scalar_type()),
        branch.defined() ? updated.data_ptr() : nullptr, quantized.data_ptr(), code_of(dtype),
        scale.data_ptr<float>(), group, rows, hidden, eps, stream_of(x)));
    return {updated, quantized, scale};
}

// The same for inputs the native path serves and calls that lose no gradient,
// else None: the auto path's common case in one call.
std::optional<std::tuple<at::Tensor, at::Tensor, at::Tensor>>
residual_rms_norm_quantized_if_supported(
    const at::Tensor& x,
    const std::optional<at::Tensor>& branch_in,
    const at::Tensor& weight,
    double eps,
    at::ScalarType dtype,
    int64_t group) {
    const at::Tensor branch = branch_in.value_or(at::Tensor());
    if (graph_recorded() || !rms_inputs_supported(x, branch, weight, eps)
        || recorded(x, branch, weight)) {
        return std::nullopt;
    }
    return residual_rms_norm_quantized(x, branch_in, weight, eps, dtype, group);
}

at::Tensor dequantize(const at::Tensor& quantized, const at::Tensor& scale, int64_t group,
                      at::ScalarType dtype) {
    TORCH_CHECK(quantized.is_cuda(), "quantized must be a HIP tensor");
    refuse_tangents("dequantize", {quantized, scale});
    refuse_recording("dequantize");
    TORCH_CHECK(scale.device() == quantized.device(),
                "all tensors must be on the same HIP device");
    TORCH_CHECK(code_type(quantized.scalar_type()), "quantized must use int8 or float8_e4m3fn");
    TORCH_CHECK(scale.scalar_type() == at::kFloat, "scale must use float32");
    TORCH_CHECK(supported_dtype(dtype), "dtype must be float32, float16 or bfloat16");
    TORCH_CHECK(quantized.dim() >= 1, "quantized must have at least one dimension");
    check_group(group);
    TORCH_CHECK(scale.sizes() == at::IntArrayRef(scale_sizes(quantized.sizes(), group)),
                "scale must have one value for each group of columns");
    c10::hip::HIPGuardMasqueradingAsCUDA guard(quantized.device());
    const auto codes = dense(quantized);
    const auto scales = dense(scale);
    auto values = empty_device_like(codes, dtype);
    if (values.numel() == 0) {
        return values;
    }
    const int64_t hidden = codes.size(-1);
    check_status(rln_dequantize(
        codes.data_ptr(), code_of(codes.scalar_type()), scales.data_ptr<float>(), group,
        values.data_ptr(), dtype_of(dtype), codes.numel() / hidden, hidden, stream_of(codes)));
    return values;
}

// The same, or None where the checks above would raise.
std::optional<at::Tensor> dequantize_if_supported(const at::Tensor& quantized,
                                                  const at::Tensor& scale, int64_t group,
                                                  at::ScalarType dtype) {
    if (graph_recorded() || !quantized.is_cuda() || scale.device() != quantized.device()
        || quantized.dim() < 1
        || !code_type(quantized.scalar_type()) || scale.scalar_type() != at::kFloat
        || quantized.size(-1) < 1
        || scale.sizes() != at::IntArrayRef(scale_sizes(quantized.sizes(), group))
        || (at::GradMode::is_enabled() && scale.requires_grad())
        || has_tangent(quantized) || has_tangent(scale)) {
        return std::nullopt;
    }
    return dequantize(quantized, scale, group, dtype);
}

}  // namespace

void bind_rms(pybind11::module_& module) {
    module.def("residual_rms_norm", &residual_rms_norm);
    module.def("residual_rms_norm_if_supported", &residual_rms_norm_if_supported);
    module.def("rms_inputs_supported",
               [](const at::Tensor& x, const std::optional<at::Tensor>& branch,
                  const at::Tensor& weight, double eps) {
                   return rms_inputs_supported(x, branch.value_or(at::Tensor()), weight, eps);
               });
    module.def("residual_rms_norm_forward", &residual_rms_norm_forward);
    module.def("residual_rms_norm_backward", &residual_rms_norm_backward);
    module.def("residual_rms_norm_quantized", &residual_rms_norm_quantized);
    module.def("residual_rms_norm_quantized_if_supported",
               &residual_rms_norm_quantized_if_supported);
    module.def("dequantize", &dequantize);
    module.def("dequantize_if_supported", &dequantize_if_supported);
}
