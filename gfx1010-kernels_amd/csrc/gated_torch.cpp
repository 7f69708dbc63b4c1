// PyTorch glue for the gated residual norm's C ABI (include/rln.h, rln_gated_*);
// part of the module `gfx1010_kernels._C`:
//
//   gated_residual_rms_norm(x, branch, weight, branch_weight, gate, eps, branch_eps,
//                           residual_scale, branch_scale, normalized_dtype)
//       autograd op returning (updated, normalized)
//   gated_residual_rms_norm_if_supported(...)   the same, or None
//   gated_inputs_refusal(...)                   why the kernels refuse the inputs, or None
//   gated_residual_rms_norm_forward(...)        (updated, normalized, statistics)
//   gated_residual_rms_norm_backward(...)       the five gradients, None where not asked
//
// The reference has no such operator.

#include "node_torch.h"

#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>

#include <cmath>
#include <optional>
#include <tuple>

using namespace rln_glue;

namespace {

using OptionalTensor = std::optional<at::Tensor>;

constexpr const char* kWhat = "gated residual RMSNorm";

// A gate or weight over x's rows: the rows that share one row of it, or 0 where
// its shape does not repeat over whole runs of x's rows. Its leading dimensions are
// x's from the first on, and 1 (or missing, on the left) from some dimension on.
int64_t factor_rows(const at::Tensor& factor, const at::Tensor& x) {
    const int64_t dims = x.dim();
    const int64_t missing = dims - factor.dim();
    if (factor.dim() < 1 || missing < 0 || factor.size(-1) != x.size(-1)) {
        return 0;
    }
    const auto size = [&](int64_t i) { return i < missing ? 1 : factor.size(i - missing); };
    int64_t rows = 1;
    int64_t i = dims - 2;
    for (; i >= 0 && size(i) == 1; --i) {
        rows *= x.size(i);
    }
    for (; i >= 0; --i) {
        if (size(i) != x.size(i)) {
            return 0;
        }
    }
    return rows;
}

// Whether the sums of both factors' gradients can be taken over the same runs.
bool factors_agree(int64_t gate_rows, int64_t weight_rows, int64_t rows) {
    return gate_rows <= 1 || gate_rows >= rows || weight_rows >= rows || gate_rows == weight_rows;
}

struct Inputs {
    const at::Tensor& x;
    const at::Tensor& branch;
    const at::Tensor& weight;
    const at::Tensor& branch_weight;  // undefined without a norm of the branch
    const at::Tensor& gate;           // undefined without a gate
    double eps;
    double branch_eps;
    double residual_scale;
    double branch_scale;
};

// Why the kernels cannot serve the inputs, or null. A message of the checks.
const char* refusal(const Inputs& in) {
    for (const at::Tensor* tensor : {&in.x, &in.branch, &in.weight, &in.branch_weight, &in.gate}) {
        if (!tensor->defined()) {
            continue;
        }
        if (!tensor->is_cuda()) {
            return "all tensors must be HIP tensors";
        }
        if (tensor->device() != in.x.device()) {
            return "all tensors must be on the same HIP device";
        }
        if (!supported_dtype(tensor->scalar_type())) {
            return "all tensors must use float16, bfloat16 or float32";
        }
        if (has_tangent(*tensor)) {
            return "the operator has no native forward-mode derivative";
        }
    }
    if (in.x.dim() < 1 || in.branch.sizes() != in.x.sizes()) {
        return "x and branch must have the same shape with at least one dimension";
    }
    const int64_t hidden = in.x.size(-1);
    if (!rln_rms_hidden_supported(hidden)) {
        return "unsupported RMSNorm hidden size: 1 to 16384 are supported";
    }
    if (in.branch_weight.defined() && in.branch_weight.sizes() != at::IntArrayRef({hidden})) {
        return "branch_weight must match the hidden size";
    }
    const int64_t rows = in.x.numel() / hidden;
    if (rows > 0) {
        const int64_t weight_rows = factor_rows(in.weight, in.x);
        const int64_t gate_rows = in.gate.defined() ? factor_rows(in.gate, in.x) : rows;
        if (weight_rows == 0 || gate_rows == 0) {
            return "gate and weight must repeat over the last of x's leading dimensions";
        }
        if (!factors_agree(gate_rows, weight_rows, rows)) {
            return "gate and weight must repeat over the same rows";
        }
    } else if (in.weight.dim() < 1 || in.weight.size(-1) != hidden
               || (in.gate.defined() && (in.gate.dim() < 1 || in.gate.size(-1) != hidden))) {
        return "gate and weight must match the hidden size";
    }
    if (!(in.eps >= 0.0) || !(in.branch_eps >= 0.0)) {
        return "eps must not be negative";
    }
    if (!std::isfinite(in.residual_scale) || !std::isfinite(in.branch_scale)) {
        return "residual_scale and branch_scale must be finite";
    }
    return nullptr;
}

void check_inputs(const Inputs& in) {
    refuse_recording(kWhat);
    const char* why = refusal(in);
    TORCH_CHECK(why == nullptr, kWhat, ": ", why);
}

const void* data_or_null(const at::Tensor& tensor) {
    return tensor.defined() ? tensor.data_ptr() : nullptr;
}

int dtype_or_float(const at::Tensor& tensor) {
    return tensor.defined() ? dtype_of(tensor.scalar_type()) : RLN_DTYPE_F32;
}

// `kept` holds the rows that the factor points into.
rln_factor_t factor_of(const at::Tensor& factor, const at::Tensor& x, at::Tensor* kept) {
    rln_factor_t out{};
    if (factor.defined()) {
        *kept = as_rows(factor, &out.stride);
        out.data = kept->data_ptr();
        out.dtype = dtype_of(factor.scalar_type());
        out.rows = factor_rows(factor, x);
    }
    return out;
}

// statistics, when given, receives what the backward needs.
std::tuple<at::Tensor, at::Tensor> forward_impl(
    const Inputs& in, std::optional<at::ScalarType> normalized_dtype, at::Tensor* statistics) {
    check_inputs(in);
    const at::ScalarType output_type = normalized_dtype.value_or(in.x.scalar_type());
    TORCH_CHECK(supported_dtype(output_type),
                "normalized_dtype must be float32, float16 or bfloat16");
    c10::hip::HIPGuardMasqueradingAsCUDA guard(in.x.device());
    const int64_t hidden = in.x.size(-1);
    const int64_t rows = in.x.numel() / hidden;
    auto updated = output_like(in.x, in.x.scalar_type());
    auto normalized = output_like(in.x, output_type);
    if (statistics != nullptr) {
        *statistics = empty_device({(in.branch_weight.defined() ? 2 : 1) * rows}, at::kFloat,
                                   in.x.device());
    }
    if (rows == 0) {
        return {updated, normalized};
    }
    int64_t x_stride = 0;
    int64_t branch_stride = 0;
    const auto x = as_rows(in.x, &x_stride);
    const auto branch = as_rows(in.branch, &branch_stride);
    const auto branch_weight = dense(in.branch_weight);
    at::Tensor gate_kept;
    at::Tensor weight_kept;
    const rln_factor_t gate = factor_of(in.gate, in.x, &gate_kept);
    const rln_factor_t weight = factor_of(in.weight, in.x, &weight_kept);
    check_status(rln_gated_forward(
        x.data_ptr(), dtype_of(x.scalar_type()), x_stride, branch.data_ptr(),
        dtype_of(branch.scalar_type()), branch_stride, data_or_null(branch_weight),
        dtype_or_float(branch_weight), &gate, &weight, updated.data_ptr(), normalized.data_ptr(),
        dtype_of(output_type), statistics != nullptr ? statistics->data_ptr<float>() : nullptr,
        rows, hidden, in.residual_scale, in.branch_scale, in.eps, in.branch_eps,
        stream_of(in.x)));
    return {updated, normalized};
}

// Gradients of x, branch, weight, branch_weight and gate; `needed` as Held's.
std::vector<at::Tensor> backward_impl(
    const at::Tensor& grad_updated_in, const at::Tensor& grad_normalized_in,
    const at::Tensor& updated_in, const at::Tensor& branch_in, const at::Tensor& weight_in,
    const at::Tensor& branch_weight_in, const at::Tensor& gate_in, const at::Tensor& statistics,
    double residual_scale, double branch_scale, int64_t needed) {
    refuse_recording("gated residual RMSNorm's backward");
    refuse_tangents(kWhat, {grad_updated_in, grad_normalized_in, updated_in, branch_in, weight_in,
                            branch_weight_in, gate_in});
    // The forward's checks, with updated for x.
    const char* why = refusal(Inputs{updated_in, branch_in, weight_in, branch_weight_in, gate_in,
                                     0.0, 0.0, residual_scale, branch_scale});
    TORCH_CHECK(why == nullptr, kWhat, "'s backward: ", why);
    const auto device = updated_in.device();
    const at::ScalarType x_type = updated_in.scalar_type();
    for (const at::Tensor* grad : {&grad_updated_in, &grad_normalized_in}) {
        TORCH_CHECK(!grad->defined()
                        || (grad->device() == device && grad->sizes() == updated_in.sizes()
                            && supported_dtype(grad->scalar_type())),
                    "the upstream gradients must match updated's shape and device and use "
                    "float16, bfloat16 or float32");
    }
    TORCH_CHECK(!grad_updated_in.defined() || grad_updated_in.scalar_type() == x_type,
                "grad_updated must use x's type");
    const int64_t hidden = updated_in.size(-1);
    const int64_t rows = updated_in.numel() / hidden;
    TORCH_CHECK(statistics.scalar_type() == at::kFloat && statistics.device() == device
                    && statistics.is_contiguous()
                    && statistics.numel() == (branch_weight_in.defined() ? 2 : 1) * rows,
                "statistics are not the forward's");
    c10::hip::HIPGuardMasqueradingAsCUDA guard(device);
    const auto wants = [needed](int input) { return (needed >> input & 1) != 0; };
    const auto like = [&](const at::Tensor& tensor, bool wanted) {
        if (!wanted || !tensor.defined()) {
            return at::Tensor();
        }
        return rows == 0 ? at::zeros(tensor.sizes(), tensor.options())
                         : empty_device(tensor.sizes(), tensor.scalar_type(), device);
    };
    auto grad_x = empty_device(updated_in.sizes(), x_type, device);
    auto grad_branch = empty_device(updated_in.sizes(), branch_in.scalar_type(), device);
    // Without the norm's gradient its weight has none.
    auto grad_weight = like(weight_in, wants(2) && grad_normalized_in.defined());
    auto grad_branch_weight = like(branch_weight_in, wants(3));
    auto grad_gate = like(gate_in, wants(4));
    if (rows == 0) {
        return {grad_x, grad_branch, grad_weight, grad_branch_weight, grad_gate};
    }
    const auto updated = dense(updated_in);
    const auto grad_updated = dense(grad_updated_in);
    const auto grad_normalized = dense(grad_normalized_in);
    const auto branch_weight = dense(branch_weight_in);
    int64_t branch_stride = 0;
    const auto branch = as_rows(branch_in, &branch_stride);
    at::Tensor gate_kept;
    at::Tensor weight_kept;
    const rln_factor_t gate = factor_of(gate_in, updated, &gate_kept);
    const rln_factor_t weight = factor_of(weight_in, updated, &weight_kept);
    at::Tensor workspace;
    size_t bytes = 0;
    if (grad_weight.defined() || grad_branch_weight.defined()
        || (grad_gate.defined() && gate.rows > 1)) {
        bytes = rln_gated_backward_workspace_bytes(
            rows, hidden, dtype_of(x_type), gate.data != nullptr ? gate.rows : rows, weight.rows);
        workspace = empty_device({static_cast<int64_t>(bytes)}, at::kByte, device);
    }
    const auto output = [](at::Tensor& tensor) {
        return tensor.defined() ? tensor.data_ptr() : nullptr;
    };
    check_status(rln_gated_backward(
        data_or_null(grad_updated), data_or_null(grad_normalized),
        dtype_or_float(grad_normalized), updated.data_ptr(), dtype_of(x_type), branch.data_ptr(),
        dtype_of(branch.scalar_type()), branch_stride, data_or_null(branch_weight),
        dtype_or_float(branch_weight), &gate, &weight, statistics.data_ptr<float>(),
        grad_x.data_ptr(), grad_branch.data_ptr(), output(grad_gate), output(grad_branch_weight),
        output(grad_weight), rows, hidden, residual_scale, branch_scale, output(workspace), bytes,
        stream_of(updated)));
    return {grad_x, grad_branch, grad_weight, grad_branch_weight, grad_gate};
}

struct GatedOperator {
    static constexpr const char* name = "GatedResidualRmsNormBackward";
    static constexpr size_t inputs = 5;

    // held: updated, branch, weight, branch_weight, gate, statistics; the two scales.
    static torch::autograd::variable_list gradients(const torch::autograd::variable_list& grads,
                                                    const Held& held) {
        const auto& t = held.tensors;
        return backward_impl(grads[0], grads[1], t[0], t[1], t[2], t[3], t[4], t[5],
                             held.numbers[0], held.numbers[1], held.needed);
    }
};

bool recorded(const Inputs& in) {
    if (!at::GradMode::is_enabled()) {
        return false;
    }
    for (const at::Tensor* tensor : {&in.x, &in.branch, &in.weight, &in.branch_weight, &in.gate}) {
        if (tensor->defined() && tensor->requires_grad()) {
            return true;
        }
    }
    return false;
}

std::tuple<at::Tensor, at::Tensor> run(const Inputs& in,
                                       std::optional<at::ScalarType> normalized_dtype) {
    if (!recorded(in)) {
        return forward_impl(in, normalized_dtype, nullptr);
    }
    at::Tensor statistics;
    at::Tensor updated;
    at::Tensor normalized;
    {
        // The kernels' own outputs; nothing inside records a graph.
        at::AutoDispatchBelowADInplaceOrView below;
        std::tie(updated, normalized) = forward_impl(in, normalized_dtype, &statistics);
    }
    auto node = make_node<GatedOperator>();
    node->set_next_edges(torch::autograd::collect_next_edges(in.x, in.branch, in.weight,
                                                             in.branch_weight, in.gate));
    torch::autograd::set_history(updated, node);
    torch::autograd::set_history(normalized, node);
    node->save(updated, true);
    node->save(in.branch);
    node->save(in.weight);
    node->save(in.branch_weight);
    node->save(in.gate);
    node->save(statistics);
    node->numbers = {in.residual_scale, in.branch_scale};
    return {updated, normalized};
}

at::Tensor or_undefined(const OptionalTensor& tensor) {
    return tensor.value_or(at::Tensor());
}

}  // namespace

void bind_gated(pybind11::module_& module) {
    module.def("gated_residual_rms_norm",
               [](const at::Tensor& x, const at::Tensor& branch, const at::Tensor& weight,
                  const OptionalTensor& branch_weight, const OptionalTensor& gate, double eps,
                  double branch_eps, double residual_scale, double branch_scale,
                  std::optional<at::ScalarType> normalized_dtype) {
                   const auto post = or_undefined(branch_weight);
                   const auto gates = or_undefined(gate);
                   return run(Inputs{x, branch, weight, post, gates, eps, branch_eps,
                                     residual_scale, branch_scale}, normalized_dtype);
               });
    module.def("gated_residual_rms_norm_if_supported",
               [](const at::Tensor& x, const at::Tensor& branch, const at::Tensor& weight,
                  const OptionalTensor& branch_weight, const OptionalTensor& gate, double eps,
                  double branch_eps, double residual_scale, double branch_scale,
                  std::optional<at::ScalarType> normalized_dtype)
                   -> std::optional<std::tuple<at::Tensor, at::Tensor>> {
                   const auto post = or_undefined(branch_weight);
                   const auto gates = or_undefined(gate);
                   const Inputs in{x, branch, weight, post, gates, eps, branch_eps,
                                   residual_scale, branch_scale};
                   if (graph_recorded() || refusal(in) != nullptr) {
                       return std::nullopt;
                   }
                   return run(in, normalized_dtype);
               });
    module.def("gated_inputs_refusal",
               [](const at::Tensor& x, const at::Tensor& branch, const at::Tensor& weight,
                  const OptionalTensor& branch_weight, const OptionalTensor& gate, double eps,
                  double branch_eps, double residual_scale, double branch_scale)
                   -> std::optional<std::string> {
                   const auto post = or_undefined(branch_weight);
                   const auto gates = or_undefined(gate);
                   const char* why = refusal(Inputs{x, branch, weight, post, gates, eps,
                                                    branch_eps, residual_scale, branch_scale});
                   return why == nullptr ? std::nullopt : std::optional<std::string>(why);
               });
    // The pieces of the autograd op, for the registered custom ops.
    module.def("gated_residual_rms_norm_forward",
               [](const at::Tensor& x, const at::Tensor& branch, const at::Tensor& weight,
                  const OptionalTensor& branch_weight, const OptionalTensor& gate, double eps,
                  double branch_eps, double residual_scale, double branch_scale,
                  std::optional<at::ScalarType> normalized_dtype) {
                   const auto post = or_undefined(branch_weight);
                   const auto gates = or_undefined(gate);
                   at::Tensor statistics;
                   auto [updated, normalized] =
                       forward_impl(Inputs{x, branch, weight, post, gates, eps, branch_eps,
                                           residual_scale, branch_scale},
                                    normalized_dtype, &statistics);
                   return std::make_tuple(updated, normalized, statistics);
               });
    module.def("gated_residual_rms_norm_backward",
               [](const OptionalTensor& grad_updated, const OptionalTensor& grad_normalized,
                  const at::Tensor& updated, const at::Tensor& branch, const at::Tensor& weight,
                  const OptionalTensor& branch_weight, const OptionalTensor& gate,
                  const at::Tensor& statistics, double residual_scale, double branch_scale,
                  int64_t needed) {
                   return backward_impl(or_undefined(grad_updated), or_undefined(grad_normalized),
                                        updated, branch, weight, or_undefined(branch_weight),
                                        or_undefined(gate), statistics, residual_scale,
                                        branch_scale, needed);
               });
}
