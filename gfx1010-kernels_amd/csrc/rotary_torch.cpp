// PyTorch glue for the rotary norm of heads (include/rln.h, rln_rotary_*); part of
// the module `gfx1010_kernels._C`:
//
//   rms_norm_rotary(q, k, positions, frequencies, sections, cyclic, interleaved,
//                   q_weight, k_weight, eps)
//       autograd op returning (q, k); k is None without one
//   rms_norm_rotary_if_supported(...)   the same, or None
//   rotary_inputs_refusal(...)          why not, or None
//   rms_norm_rotary_forward(...)        (q, k) without a graph
//   rms_norm_rotary_backward(...)       gradients of q, k, q_weight, k_weight
//
// The reference has no such operator.

#include "node_torch.h"

#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>

#include <algorithm>
#include <optional>
#include <tuple>

using namespace rln_glue;

namespace {

using OptionalTensor = std::optional<at::Tensor>;

constexpr const char* kWhat = "rotary RMSNorm";
constexpr int64_t kMaxSize = 256;
constexpr int64_t kMaxHeads = 1 << 16;

struct Inputs {
    const at::Tensor& q;
    const at::Tensor& k;  // undefined where there is none
    const at::Tensor& positions;
    const at::Tensor& frequencies;
    const std::vector<int64_t>& sections;  // empty: one axis, without a dimension for it
    bool cyclic;
    bool interleaved;
    const at::Tensor& q_weight;
    const at::Tensor& k_weight;
    double eps;
};

// The dimensions of heads in front of [heads, size].
at::IntArrayRef leading(const at::Tensor& heads) {
    return heads.sizes().slice(0, heads.dim() - 2);
}

bool broadcasts(at::IntArrayRef from, at::IntArrayRef to) {
    if (from.size() > to.size()) {
        return false;
    }
    const size_t missing = to.size() - from.size();
    for (size_t i = 0; i < from.size(); ++i) {
        if (from[i] != 1 && from[i] != to[missing + i]) {
            return false;
        }
    }
    return true;
}

// Why the kernels cannot serve the inputs, or null.
const char* refusal(const Inputs& in) {
    if (in.q.dim() < 2 || (in.k.defined() && in.k.dim() < 2)) {
        return "q and k must have the dimensions [..., heads, size]";
    }
    for (const at::Tensor* tensor :
         {&in.q, &in.k, &in.positions, &in.frequencies, &in.q_weight, &in.k_weight}) {
        if (!tensor->defined()) {
            continue;
        }
        if (!tensor->is_cuda()) {
            return "all tensors must be HIP tensors";
        }
        if (tensor->device() != in.q.device()) {
            return "all tensors must be on the same HIP device";
        }
        if (has_tangent(*tensor)) {
            return "the operator has no native forward-mode derivative";
        }
    }
    const int64_t size = in.q.size(-1);
    if (size < 1 || size > kMaxSize) {
        return "heads must have 1 to 256 values";
    }
    if (!supported_dtype(in.q.scalar_type())
        || (in.k.defined() && in.k.scalar_type() != in.q.scalar_type())) {
        return "q and k must use one type of float16, bfloat16 and float32";
    }
    if (in.k.defined() && (leading(in.k) != leading(in.q) || in.k.size(-1) != size)) {
        return "q and k must have the same tokens and head size";
    }
    if (in.q.size(-2) > kMaxHeads || (in.k.defined() && in.k.size(-2) > kMaxHeads)) {
        return "at most 65536 heads are supported";
    }
    for (const at::Tensor* weight : {&in.q_weight, &in.k_weight}) {
        if (weight->defined()
            && (!supported_dtype(weight->scalar_type())
                || weight->sizes() != at::IntArrayRef({size}))) {
            return "q_weight and k_weight must have the head size and use float16, bfloat16 or "
                   "float32";
        }
    }
    if (in.k_weight.defined() && !in.k.defined()) {
        return "k_weight needs k";
    }
    const auto frequency_type = in.frequencies.scalar_type();
    if (in.frequencies.dim() != 1 || in.frequencies.size(0) < 1
        || 2 * in.frequencies.size(0) > size
        || (frequency_type != at::kFloat && frequency_type != at::kDouble)) {
        return "inverse_frequencies must hold 1 to size / 2 values in float32 or float64";
    }
    const auto position_type = in.positions.scalar_type();
    if (position_type != at::kLong && position_type != at::kInt && position_type != at::kFloat) {
        return "positions must use int64, int32 or float32";
    }
    at::IntArrayRef tokens = in.positions.sizes();
    if (!in.sections.empty()) {
        int64_t total = 0;
        for (const int64_t section : in.sections) {
            if (section < 0) {
                return "sections must not be negative";
            }
            // One that is too many alone counts as that, so that no sum wraps round.
            total += std::min(section, in.frequencies.size(0) + 1);
        }
        if (in.sections.size() > 4 || total != in.frequencies.size(0)) {
            return "sections must be 1 to 4 numbers of pairs that add up to inverse_frequencies";
        }
        if (tokens.empty() || tokens[0] != static_cast<int64_t>(in.sections.size())) {
            return "positions must have one row for each section";
        }
        tokens = tokens.slice(1);
    }
    if (!broadcasts(tokens, leading(in.q))) {
        return "positions must broadcast over the tokens";
    }
    if (at::GradMode::is_enabled()
        && (in.positions.requires_grad() || in.frequencies.requires_grad())) {
        return "positions and inverse_frequencies have no gradient";
    }
    if (in.q.numel() / size > 0 && in.q.numel() / size / in.q.size(-2) > INT32_MAX / 2) {
        return "too many tokens";
    }
    if (!(in.eps >= 0.0)) {
        return "eps must not be negative";
    }
    return nullptr;
}

void check_inputs(const Inputs& in) {
    refuse_recording(kWhat);
    const char* why = refusal(in);
    TORCH_CHECK(why == nullptr, kWhat, ": ", why);
}

// Heads as [outer, inner, heads, size] with consecutive elements: views where the
// strides allow it, copies elsewhere.
at::Tensor as_heads(const at::Tensor& heads) {
    at::Tensor out = stored(heads);
    if (out.size(-1) != 1 && out.stride(-1) != 1) {
        out = out.contiguous();
    }
    while (out.dim() < 4) {
        out = out.unsqueeze(0);
    }
    return out.dim() == 4 ? out : out.flatten(0, -4);
}

rln_heads_t heads_of(const at::Tensor& heads) {
    return rln_heads_t{heads.data_ptr(), heads.stride(0), heads.stride(1), heads.stride(2)};
}

// The tables of a call and what they point to.
struct Rotary {
    rln_rotary_t table;
    std::vector<uint8_t> axes;
    at::Tensor positions;
    at::Tensor frequencies;
    int64_t outer;
    int64_t inner;
};

// `lead`: the heads' leading dimensions.
void fill_rotary(const Inputs& in, at::IntArrayRef lead, Rotary* out) {
    const int64_t axes = in.sections.empty() ? 1 : static_cast<int64_t>(in.sections.size());
    std::vector<int64_t> sizes{axes};
    sizes.insert(sizes.end(), lead.begin(), lead.end());
    at::Tensor positions = stored(in.positions);
    if (in.sections.empty()) {
        positions = positions.unsqueeze(0);
    }
    // The axes stay in front of tokens that broadcast.
    while (positions.dim() < static_cast<int64_t>(sizes.size())) {
        positions = positions.unsqueeze(1);
    }
    positions = positions.expand(sizes);
    while (positions.dim() < 3) {
        positions = positions.unsqueeze(1);
    }
    if (positions.dim() > 3) {
        positions = positions.flatten(1, -2);
    }
    out->positions = positions;
    out->frequencies = dense(in.frequencies);
    out->outer = positions.size(1);
    out->inner = positions.size(2);
    const int64_t pairs = in.frequencies.size(0);
    out->axes.assign(pairs, 0);
    if (in.cyclic) {
        for (int64_t axis = 1; axis < axes; ++axis) {
            for (int64_t turn = 0; turn < in.sections[axis] && axis + turn * axes < pairs; ++turn) {
                out->axes[axis + turn * axes] = static_cast<uint8_t>(axis);
            }
        }
    } else {
        int64_t pair = 0;
        for (int64_t axis = 0; axis < axes && !in.sections.empty(); ++axis) {
            for (int64_t i = 0; i < in.sections[axis]; ++i) {
                out->axes[pair++] = static_cast<uint8_t>(axis);
            }
        }
    }
    rln_rotary_t& table = out->table;
    table = rln_rotary_t{};
    table.positions = positions.data_ptr();
    table.positions_type = positions.scalar_type() == at::kLong ? RLN_POSITIONS_I64
        : positions.scalar_type() == at::kInt ? RLN_POSITIONS_I32 : RLN_POSITIONS_F32;
    table.axis_stride = positions.stride(0);
    table.outer_stride = positions.stride(1);
    table.token_stride = positions.stride(2);
    table.frequencies = out->frequencies.data_ptr();
    table.wide_frequencies = out->frequencies.scalar_type() == at::kDouble;
    table.axis_of_pair = out->axes.data();
    table.axes = axes;
    table.pairs = pairs;
    table.interleaved = in.interleaved;
}

// One run of tokens where every stride allows it: the kernels then divide no
// token's number.
void merge_tokens(Rotary* rotary, std::initializer_list<rln_heads_t*> all) {
    const auto merges = [rotary](int64_t outer, int64_t token) {
        return rotary->outer == 1 || outer == token * rotary->inner;
    };
    bool one = merges(rotary->table.outer_stride, rotary->table.token_stride);
    for (const rln_heads_t* heads : all) {
        one = one && (heads->data == nullptr || merges(heads->outer_stride, heads->token_stride));
    }
    if (one) {
        rotary->inner *= rotary->outer;
        rotary->outer = 1;
    } else if (rotary->inner == 1) {  // as in a decode step: rows of one token each
        rotary->inner = rotary->outer;
        rotary->outer = 1;
        rotary->table.token_stride = rotary->table.outer_stride;
        for (rln_heads_t* heads : all) {
            heads->token_stride = heads->outer_stride;
        }
    }
}

const void* data_or_null(const at::Tensor& tensor) {
    return tensor.defined() ? tensor.data_ptr() : nullptr;
}

int dtype_or_float(const at::Tensor& tensor) {
    return tensor.defined() ? dtype_of(tensor.scalar_type()) : RLN_DTYPE_F32;
}

std::tuple<at::Tensor, at::Tensor> forward_impl(const Inputs& in) {
    check_inputs(in);
    c10::hip::HIPGuardMasqueradingAsCUDA guard(in.q.device());
    const auto type = in.q.scalar_type();
    auto q_out = output_like(in.q, type);
    auto k_out = in.k.defined() ? output_like(in.k, type) : at::Tensor();
    if (q_out.numel() == 0 && (!k_out.defined() || k_out.numel() == 0)) {
        return {q_out, k_out};
    }
    Rotary rotary;
    fill_rotary(in, leading(in.q), &rotary);
    rln_rotary_side_t sides[2] = {};
    at::Tensor kept[2];
    at::Tensor weights[2];
    const at::Tensor* heads[2] = {&in.q, &in.k};
    const at::Tensor* given[2] = {&in.q_weight, &in.k_weight};
    at::Tensor* outputs[2] = {&q_out, &k_out};
    for (int i = 0; i < 2; ++i) {
        if (!heads[i]->defined() || heads[i]->numel() == 0) {
            continue;
        }
        kept[i] = as_heads(*heads[i]);
        weights[i] = dense(*given[i]);
        sides[i].heads = heads_of(kept[i]);
        sides[i].count = kept[i].size(2);
        sides[i].weight = data_or_null(weights[i]);
        sides[i].weight_dtype = dtype_or_float(weights[i]);
        sides[i].output = outputs[i]->data_ptr();
    }
    merge_tokens(&rotary, {&sides[0].heads, &sides[1].heads});
    check_status(rln_rotary_forward(&sides[0], &sides[1], dtype_of(type), &rotary.table,
                                    rotary.outer, rotary.inner, in.q.size(-1), in.eps,
                                    stream_of(in.q)));
    return {q_out, k_out};
}

// Gradients of q, k, q_weight and k_weight; those of a side whose upstream gradient
// is undefined are undefined. q and k are read where they have a norm.
std::vector<at::Tensor> backward_impl(
    const at::Tensor& grad_q, const at::Tensor& grad_k, const at::Tensor& q, const at::Tensor& k,
    const at::Tensor& positions, const at::Tensor& frequencies,
    const std::vector<int64_t>& sections, bool cyclic, bool interleaved,
    const at::Tensor& q_weight, const at::Tensor& k_weight, double eps, int64_t needed) {
    refuse_recording("rotary RMSNorm's backward");
    std::vector<at::Tensor> results(4);
    const at::Tensor* grads[2] = {&grad_q, &grad_k};
    const at::Tensor* heads[2] = {&q, &k};
    const at::Tensor* given[2] = {&q_weight, &k_weight};
    const at::Tensor none;
    const at::Tensor& first = grad_q.defined() ? grad_q : grad_k;
    if (!first.defined()) {
        return results;
    }
    // The forward's checks, with the gradients for the heads.
    const at::Tensor& second = grad_q.defined() ? grad_k : none;
    const Inputs in{first, second, positions, frequencies, sections, cyclic, interleaved,
                    grad_q.defined() ? q_weight : k_weight,
                    second.defined() ? k_weight : none, eps};
    const char* why = refusal(in);
    TORCH_CHECK(why == nullptr, kWhat, "'s backward: ", why);
    const auto device = first.device();
    const auto type = first.scalar_type();
    const int64_t size = first.size(-1);
    c10::hip::HIPGuardMasqueradingAsCUDA guard(device);
    Rotary rotary;
    fill_rotary(in, leading(first), &rotary);
    rln_rotary_side_t sides[2] = {};
    at::Tensor kept[2][2];
    at::Tensor weights[2];
    bool sums = false;
    for (int i = 0; i < 2; ++i) {
        const at::Tensor& grad = *grads[i];
        if (!grad.defined()) {
            continue;
        }
        const bool normed = given[i]->defined();
        TORCH_CHECK(!normed
                        || (heads[i]->defined() && heads[i]->device() == device
                            && heads[i]->scalar_type() == type && heads[i]->sizes() == grad.sizes()
                            && !has_tangent(*heads[i])),
                    kWhat, "'s backward: the heads must match their gradient");
        results[i] = empty_device(grad.sizes(), type, device);
        const bool sum = normed && (needed >> (2 + i) & 1) != 0;
        if (sum) {
            results[2 + i] = grad.numel() == 0
                ? at::zeros({size}, given[i]->options())
                : empty_device({size}, given[i]->scalar_type(), device);
        }
        if (grad.numel() == 0) {
            continue;
        }
        kept[i][0] = as_heads(grad);
        sides[i].grad = heads_of(kept[i][0]);
        sides[i].count = kept[i][0].size(2);
        sides[i].output = results[i].data_ptr();
        if (normed) {
            kept[i][1] = as_heads(*heads[i]);
            weights[i] = dense(*given[i]);
            sides[i].heads = heads_of(kept[i][1]);
            sides[i].weight = weights[i].data_ptr();
            sides[i].weight_dtype = dtype_of(weights[i].scalar_type());
            sides[i].grad_weight = sum ? results[2 + i].data_ptr() : nullptr;
            sums = sums || sum;
        }
    }
    if (sides[0].count == 0 && sides[1].count == 0) {
        return results;
    }
    merge_tokens(&rotary, {&sides[0].heads, &sides[1].heads, &sides[0].grad, &sides[1].grad});
    at::Tensor workspace;
    size_t bytes = 0;
    if (sums) {
        bytes = rln_rotary_backward_workspace_bytes(rotary.outer, rotary.inner, sides[0].count,
                                                    sides[1].count, size, rotary.table.pairs,
                                                    dtype_of(type));
        workspace = empty_device({static_cast<int64_t>(bytes)}, at::kByte, device);
    }
    check_status(rln_rotary_backward(&sides[0], &sides[1], dtype_of(type), &rotary.table,
                                     rotary.outer, rotary.inner, size, eps,
                                     workspace.defined() ? workspace.data_ptr() : nullptr, bytes,
                                     stream_of(first)));
    return results;
}

struct RotaryOperator {
    static constexpr const char* name = "RmsNormRotaryBackward";
    static constexpr size_t inputs = 4;

    // held: q, k (where they have a norm), positions, frequencies, q_weight, k_weight;
    // cyclic, interleaved, the sections; eps.
    static torch::autograd::variable_list gradients(const torch::autograd::variable_list& grads,
                                                    const Held& held) {
        const auto& t = held.tensors;
        const std::vector<int64_t> sections(held.integers.begin() + 2, held.integers.end());
        return backward_impl(grads[0], grads.size() > 1 ? grads[1] : at::Tensor(), t[0], t[1],
                             t[2], t[3], sections, held.integers[0] != 0, held.integers[1] != 0,
                             t[4], t[5], held.numbers[0], held.needed);
    }
};

bool recorded(const Inputs& in) {
    if (!at::GradMode::is_enabled()) {
        return false;
    }
    for (const at::Tensor* tensor : {&in.q, &in.k, &in.q_weight, &in.k_weight}) {
        if (tensor->defined() && tensor->requires_grad()) {
            return true;
        }
    }
    return false;
}

std::tuple<at::Tensor, OptionalTensor> run(const Inputs& in) {
    const auto optional = [](const at::Tensor& tensor) {
        return tensor.defined() ? OptionalTensor(tensor) : std::nullopt;
    };
    if (!recorded(in)) {
        auto [q, k] = forward_impl(in);
        return {q, optional(k)};
    }
    at::Tensor q;
    at::Tensor k;
    {
        // The kernels' own outputs; nothing inside records a graph.
        at::AutoDispatchBelowADInplaceOrView below;
        std::tie(q, k) = forward_impl(in);
    }
    auto node = make_node<RotaryOperator>();
    node->set_next_edges(
        torch::autograd::collect_next_edges(in.q, in.k, in.q_weight, in.k_weight));
    torch::autograd::set_history(q, node);
    if (k.defined()) {
        torch::autograd::set_history(k, node);
    }
    node->save(in.q_weight.defined() ? in.q : at::Tensor());
    node->save(in.k_weight.defined() ? in.k : at::Tensor());
    node->save(in.positions);
    node->save(in.frequencies);
    node->save(in.q_weight);
    node->save(in.k_weight);
    node->integers = {in.cyclic, in.interleaved};
    node->integers.insert(node->integers.end(), in.sections.begin(), in.sections.end());
    node->numbers = {in.eps};
    return {q, optional(k)};
}

at::Tensor or_undefined(const OptionalTensor& tensor) {
    return tensor.value_or(at::Tensor());
}

// Calls `use` with the arguments as Inputs.
template <typename Use>
auto with_inputs(const Use& use) {
    return [use](const at::Tensor& q, const OptionalTensor& k, const at::Tensor& positions,
                 const at::Tensor& frequencies, const std::vector<int64_t>& sections, bool cyclic,
                 bool interleaved, const OptionalTensor& q_weight, const OptionalTensor& k_weight,
                 double eps) {
        const auto keys = or_undefined(k);
        const auto q_own = or_undefined(q_weight);
        const auto k_own = or_undefined(k_weight);
        return use(Inputs{q, keys, positions, frequencies, sections, cyclic, interleaved, q_own,
                          k_own, eps});
    };
}

}  // namespace

void bind_rotary(pybind11::module_& module) {
    module.def("rms_norm_rotary", with_inputs([](const Inputs& in) { return run(in); }));
    module.def("rms_norm_rotary_if_supported",
               with_inputs([](const Inputs& in)
                               -> std::optional<std::tuple<at::Tensor, OptionalTensor>> {
                   if (graph_recorded() || refusal(in) != nullptr) {
                       return std::nullopt;
                   }
                   return run(in);
               }));
    module.def("rotary_inputs_refusal",
               with_inputs([](const Inputs& in) -> std::optional<std::string> {
                   const char* why = refusal(in);
                   return why == nullptr ? std::nullopt : std::optional<std::string>(why);
               }));
    // The pieces of the autograd op, for the registered custom ops; an empty tensor
    // stands for no k.
    module.def("rms_norm_rotary_forward", with_inputs([](const Inputs& in) {
                   auto [q, k] = forward_impl(in);
                   return std::make_tuple(
                       q, k.defined() ? k : empty_device({0}, q.scalar_type(), q.device()));
               }));
    module.def("rms_norm_rotary_backward",
               [](const OptionalTensor& grad_q, const OptionalTensor& grad_k,
                  const OptionalTensor& q, const OptionalTensor& k, const at::Tensor& positions,
                  const at::Tensor& frequencies, const std::vector<int64_t>& sections, bool cyclic,
                  bool interleaved, const OptionalTensor& q_weight,
                  const OptionalTensor& k_weight, double eps, int64_t needed) {
                   return backward_impl(or_undefined(grad_q), or_undefined(grad_k),
                                        or_undefined(q), or_undefined(k), positions, frequencies,
                                        sections, cyclic, interleaved, or_undefined(q_weight),
                                        or_undefined(k_weight), eps, needed);
               });
}
