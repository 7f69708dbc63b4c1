// Shared by the torch glue of the C ABI (rln_torch.cpp, rms_torch.cpp, gated_torch.cpp,
// rotary_torch.cpp): status to exception, element types, and allocation.
#ifndef RLN_TORCH_H
#define RLN_TORCH_H

#include <torch/extension.h>

#include <ATen/TracerMode.h>
#include <ATen/hip/EmptyTensor.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>

#include <functional>
#include <initializer_list>

#include "rln.h"

namespace rln_glue {

inline bool supported_dtype(at::ScalarType type) {
    return type == at::kFloat || type == at::kHalf || type == at::kBFloat16;
}

inline void check_status(int status) {
    TORCH_CHECK(status == RLN_OK, rln_last_error());
}

inline int dtype_of(at::ScalarType type) {
    if (type == at::kHalf) {
        return RLN_DTYPE_F16;
    }
    if (type == at::kBFloat16) {
        return RLN_DTYPE_BF16;
    }
    return RLN_DTYPE_F32;
}

// Whether a forward-mode derivative comes with `tensor` (the one level that
// torch.autograd.forward_ad has). The kernels read addresses and know nothing of it.
inline bool has_tangent(const at::Tensor& tensor) {
    return tensor.defined() && tensor._fw_grad(/*level=*/0).defined();
}

// Raises where a forward-mode derivative would be dropped: the operators have a
// backward, and no forward derivative.
inline void refuse_tangents(
    const char* what,
    std::initializer_list<std::reference_wrapper<const at::Tensor>> tensors) {
    for (const at::Tensor& tensor : tensors) {
        TORCH_CHECK(!has_tangent(tensor), what, " has no native forward-mode derivative");
    }
}

// Whether something on this thread looks on at, or takes over, every operator:
// a TorchDispatchMode (FakeTensorMode among them), a functorch transform, a
// trace. Its dispatch key is then in the thread's included set.
inline bool dispatch_watched() {
    return !(c10::impl::tls_local_dispatch_key_set().included_ - c10::default_included_set).empty();
}

// Whether the operators called on this thread are recorded into a graph
// (torch.jit.trace, make_fx). Such a graph would hold the outputs' allocations
// and no kernel, and return memory as it comes: the calls decline or raise, and
// go through the registered operators (torch.ops.gfx1010_kernels) instead, which
// a graph holds whole. A registered operator's own kernel runs outside of the
// recording. PreDispatch stands for make_fx(pre_dispatch=True).
inline bool graph_recorded() {
    return dispatch_watched()
        && (at::tracer::impl::is_dispatch_enabled()
            || c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::PreDispatch)
            || c10::impl::TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY)
                   .has_value());
}

inline void refuse_recording(const char* what) {
    TORCH_CHECK(!graph_recorded(), what, " is being recorded into a graph that cannot hold it; "
                "torch.ops.gfx1010_kernels has the operators a graph can hold");
}

// Outputs and scratch, straight from the caching allocator. at::empty goes
// through the dispatcher and, under torch.use_deterministic_algorithms(True),
// fills every new tensor with NaN (torch.utils.deterministic.
// fill_uninitialized_memory): seven extra passes per training step over
// memory that the kernels overwrite whole. Measured on MI355X: eager forward +
// backward of [65536, 1024], fp16 branch, in deterministic mode 499.5 -> 349.9
// us; a no_grad call of [8, 768] (bound by the host) 8.40 -> 7.83 us. A watched
// thread keeps at::empty: a memory-counting mode sees the allocations, and a
// FakeTensorMode or functorch transform around tensors of real memory is
// refused as by any operator that asks for their addresses.
inline at::Tensor empty_device(at::IntArrayRef sizes, at::ScalarType type, const at::Device& device) {
    if (dispatch_watched()) {
        return at::empty(sizes, at::TensorOptions(device).dtype(type));
    }
    return at::Tensor(at::detail::empty_cuda(sizes, type, device, std::nullopt));
}

// at::empty_like of a contiguous tensor. What it takes over from `like` goes
// through it: dimension names, a __torch_dispatch__ subclass, and the strides of
// dimensions of size 1, of which contiguity says nothing, where they are not
// the plain row-major ones.
inline at::Tensor empty_device_like(const at::Tensor& like, at::ScalarType type) {
    bool plain = !dispatch_watched() && !like.has_names()
        && !like.key_set().has(c10::DispatchKey::Python);
    int64_t stride = 1;
    for (int64_t i = like.dim() - 1; plain && i >= 0; --i) {
        plain = like.stride(i) == stride;
        stride *= like.size(i);
    }
    return plain ? empty_device(like.sizes(), type, like.device())
                 : at::empty_like(like, like.options().dtype(type));
}

}  // namespace rln_glue

// The entry points of rms_torch.cpp, gated_torch.cpp and rotary_torch.cpp.
void bind_rms(pybind11::module_& module);
void bind_gated(pybind11::module_& module);
void bind_rotary(pybind11::module_& module);

#endif  // RLN_TORCH_H
