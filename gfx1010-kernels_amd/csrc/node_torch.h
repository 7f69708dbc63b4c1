// The graph node of an operator whose backward is one call of its kernels
// (gated_torch.cpp, rotary_torch.cpp): saved tensors, constants, compiled autograd and
// the refusal of second-order gradients. A node of its own instead of a
// torch::autograd::Function, for the reason given at rms_torch.cpp's node.
#ifndef NODE_TORCH_H
#define NODE_TORCH_H

#include "rows_torch.h"

#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/dynamo/compiled_autograd.h>

#include <memory>
#include <mutex>
#include <string>
#include <vector>

namespace rln_glue {

// What gradients are computed from.
struct Held {
    std::vector<at::Tensor> tensors;  // undefined where none was saved
    std::vector<int64_t> integers;
    std::vector<double> numbers;
    int64_t needed = 0;  // bit i: the gradient of input i is asked for
};

// Operator: `name` (static const char*), `gradients(grads, held)` (static).
template <typename Operator>
class KernelNode : public torch::autograd::Node {
 public:
    std::string name() const override {
        return Operator::name;
    }

    // Tensors in the order in which the gradients find them.
    void save(const at::Tensor& tensor, bool is_output = false) {
        if (tensor.defined()) {
            present_ |= int64_t{1} << count_;
            outputs_ |= static_cast<int64_t>(is_output) << count_;
            saved_.emplace_back(tensor, is_output);
        }
        ++count_;
    }

    std::vector<int64_t> integers;
    std::vector<double> numbers;

    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        for (auto& saved : saved_) {
            saved.reset_data();
        }
    }

    torch::autograd::variable_list apply(torch::autograd::variable_list&& grads) override {
        std::lock_guard<std::mutex> lock(mutex_);
        return gradients(grads, unpack());
    }

    // Compiled autograd: what the node holds, and its gradients as one call that the
    // compiled graph makes with its own tensors.
    void compiled_args(torch::dynamo::autograd::CompiledNodeArgs& args) const override {
        args.collect(present_);
        size_t next = 0;
        for (int i = 0; i < count_; ++i) {
            if (present_ >> i & 1) {
                args.collect(saved_[next++], (outputs_ >> i & 1) != 0);
            }
        }
        for (const int64_t value : integers) {
            args.collect(value);
        }
        for (const double value : numbers) {
            args.collect(value);
        }
    }

    torch::autograd::variable_list apply_with_saved(
        const torch::autograd::variable_list& grads,
        torch::dynamo::autograd::SwapSavedVariables& swap) override {
        namespace compiled = torch::dynamo::autograd;
        for (auto& saved : saved_) {
            swap.before(saved);
        }
        const Held held = unpack();
        compiled::PackedArgs packed;
        std::vector<at::TypePtr> types;
        for (const auto& tensor : held.tensors) {
            if (tensor.defined()) {
                packed.pack(tensor);
                types.push_back(compiled::IValuePacker<at::Tensor>::packed_type());
            }
        }
        for (const int64_t value : held.integers) {
            packed.pack(value);
            types.push_back(compiled::IValuePacker<int64_t>::packed_type());
        }
        for (const double value : held.numbers) {
            packed.pack(value);
            types.push_back(compiled::IValuePacker<double>::packed_type());
        }
        packed.pack(held.needed);
        types.push_back(compiled::IValuePacker<int64_t>::packed_type());
        const auto call = [present = present_, count = count_, whole = held.integers.size(),
                           real = held.numbers.size()](
                              const torch::autograd::variable_list& given_grads,
                              const std::vector<c10::IValue>& args) {
            compiled::PackedArgs given(args);
            Held inner;
            for (int i = 0; i < count; ++i) {
                inner.tensors.push_back(present >> i & 1 ? given.unpack<at::Tensor>()
                                                         : at::Tensor());
            }
            for (size_t i = 0; i < whole; ++i) {
                inner.integers.push_back(given.unpack<int64_t>());
            }
            for (size_t i = 0; i < real; ++i) {
                inner.numbers.push_back(given.unpack<double>());
            }
            inner.needed = given.unpack<int64_t>();
            return gradients(given_grads, inner);
        };
        const auto& compiler = compiled::getPyCompilerInterface();
        const std::string function = compiler->bind_function(
            swap.get_py_compiler(), name(), call, types,
            /*is_custom_function=*/true, /*is_traceable=*/false);
        auto results = compiler->call_function(
            swap.get_py_compiler(), "apply_functional", function, grads, packed.vec(),
            compiled::IValuePacker<std::vector<std::optional<torch::autograd::InputMetadata>>>::
                pack(compiled::get_input_metadata(next_edges())));
        for (auto& saved : saved_) {
            swap.after(saved);
        }
        return results;
    }

 private:
    Held unpack() {
        Held held;
        size_t next = 0;
        for (int i = 0; i < count_; ++i) {
            if (present_ >> i & 1) {
                held.tensors.push_back(
                    saved_[next++].unpack(outputs_ >> i & 1 ? getptr() : nullptr));
            } else {
                held.tensors.emplace_back();
            }
        }
        held.integers = integers;
        held.numbers = numbers;
        for (size_t input = 0; input < num_outputs(); ++input) {
            held.needed |= static_cast<int64_t>(task_should_compute_output(input)) << input;
        }
        return held;
    }

    static torch::autograd::variable_list gradients(const torch::autograd::variable_list& grads,
                                                    const Held& held) {
        bool any = false;
        for (const auto& grad : grads) {
            any = any || grad.defined();
        }
        auto results = any ? Operator::gradients(grads, held) : torch::autograd::variable_list();
        results.resize(Operator::inputs);
        if (any && at::GradMode::is_enabled()) {
            // create_graph: the gradients are constants of a backward that
            // has none of its own; differentiating them again raises.
            refuse_second_order(grads, held.tensors, results);
        }
        return results;
    }

    static void refuse_second_order(const torch::autograd::variable_list& grads,
                                    const std::vector<at::Tensor>& tensors,
                                    const torch::autograd::variable_list& results) {
        torch::autograd::variable_list given;
        for (const auto* list : {&grads, &tensors}) {
            for (const auto& tensor : *list) {
                if (tensor.defined()) {
                    given.push_back(tensor);
                }
            }
        }
        if (!torch::autograd::any_variable_requires_grad(given)) {
            return;
        }
        const auto refusal = std::make_shared<torch::autograd::NotImplemented>(
            std::string(Operator::name) + " (second-order gradients)",
            torch::autograd::collect_next_edges(given));
        for (const auto& result : results) {
            if (result.defined()) {
                torch::autograd::set_history(result, refusal);
            }
        }
    }

    std::vector<torch::autograd::SavedVariable> saved_;
    int64_t present_ = 0;
    int64_t outputs_ = 0;
    int count_ = 0;
};

template <typename Operator>
std::shared_ptr<KernelNode<Operator>> make_node() {
    return std::shared_ptr<KernelNode<Operator>>(new KernelNode<Operator>(),
                                                 torch::autograd::deleteNode);
}

}  // namespace rln_glue

#endif  // NODE_TORCH_H
