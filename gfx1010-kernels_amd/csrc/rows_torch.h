// Shared by the torch glue of the row operators (rms_torch.cpp, gated_torch.cpp,
// rotary_torch.cpp): tensors as rows at a stride, outputs like an input, streams.
#ifndef ROWS_TORCH_H
#define ROWS_TORCH_H

#include "rln_torch.h"

#include <ATen/NamedTensorUtils.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>

#include <optional>

namespace rln_glue {

// The one step between consecutive rows of `tensor` seen as [rows, hidden], or
// nullopt where its leading dimensions are no single run of rows or the elements
// of a row are apart.
inline std::optional<int64_t> row_stride(const at::Tensor& tensor) {
    const int64_t dims = tensor.dim();
    if (tensor.size(-1) != 1 && tensor.stride(-1) != 1) {
        return std::nullopt;
    }
    int64_t stride = tensor.size(-1);
    int64_t next = -1;  // the step that the dimension outside has to have
    for (int64_t i = dims - 2; i >= 0; --i) {
        if (tensor.size(i) == 1) {
            continue;
        }
        if (next < 0) {
            stride = tensor.stride(i);
        } else if (tensor.stride(i) != next) {
            return std::nullopt;
        }
        next = tensor.stride(i) * tensor.size(i);
    }
    return stride;
}

// `tensor` with its values in memory: the imaginary part of a conjugate is a view
// whose elements are negated as they are read.
inline at::Tensor stored(const at::Tensor& tensor) {
    return tensor.is_neg() ? tensor.resolve_neg() : tensor;
}

// `tensor` as one dense run of values; undefined where it is.
inline at::Tensor dense(const at::Tensor& tensor) {
    return tensor.defined() ? stored(tensor.contiguous()) : tensor;
}

// `tensor` with rows of consecutive elements one stride apart, copied only
// where it has none.
inline at::Tensor as_rows(const at::Tensor& given, int64_t* stride) {
    const auto tensor = stored(given);
    const auto found = row_stride(tensor);
    *stride = found.value_or(tensor.size(-1));
    return found ? tensor : tensor.contiguous();
}

// Dense outputs in x's shape, with its dimension names; of a contiguous x
// whatever else empty_device_like takes over.
inline at::Tensor output_like(const at::Tensor& x, at::ScalarType type) {
    if (x.is_contiguous()) {
        return empty_device_like(x, type);
    }
    auto output = empty_device(x.sizes(), type, x.device());
    if (x.has_names()) {
        at::namedinference::propagate_names(output, x);
    }
    return output;
}

inline hipStream_t stream_of(const at::Tensor& x) {
    return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(x.device().index()).stream();
}

}  // namespace rln_glue

#endif  // ROWS_TORCH_H
