// Instances of the gated residual norm's kernels (gated_device.h), one
// translation unit per stream type (RMS_STREAM: float, half_t or bf16_t) and
// pass (RMS_PASS: 1 forward, 2 backward).

#include "gated_device.h"

namespace rln {
namespace gated {
namespace {

template <typename Kernel, typename Args>
int launch(Kernel kernel, const Args& a, int64_t blocks, int threads, size_t lds,
           hipStream_t stream, const char* what) {
    kernel<<<dim3(static_cast<unsigned>(blocks)), threads, lds, stream>>>(a);
    return check_launch(what);
}

#if RMS_PASS == 1
template <typename X, typename B, int V, bool kPost>
int run(const ForwardArgs& a, const Shape& shape, hipStream_t stream) {
    auto kernel = a.words ? forward_kernel<X, B, V, kPost, Access::kWords>
                          : forward_kernel<X, B, V, kPost, Access::kElements>;
    if constexpr (V == 1) {
        if (shape.row_lanes < kWave) {
            kernel = forward_kernel<X, B, 1, kPost, Access::kLanes>;
        }
    }
    return launch(kernel, a, forward_blocks(a.rows, shape), shape.threads, 0, stream,
                  "gated forward_kernel");
}
using Args = ForwardArgs;
#else
template <typename X, typename B, int V, bool kPost, bool kToken>
int run_token(const BackwardArgs& a, const Shape& shape, hipStream_t stream) {
    constexpr int kLaneColumns = V * kColumns<X>;
    const size_t lds = kLaneColumns > 8
        ? 2 * static_cast<size_t>(shape.threads) * kLaneColumns * sizeof(float)
        : a.partials == nullptr
        ? 0 : static_cast<size_t>(teams_of(shape) - 1) * a.hidden * sizeof(float);
    auto kernel = a.words ? backward_kernel<X, B, V, kPost, kToken, Access::kWords>
                          : backward_kernel<X, B, V, kPost, kToken, Access::kElements>;
    if constexpr (V == 1) {
        if (shape.row_lanes < kWave) {
            kernel = backward_kernel<X, B, 1, kPost, kToken, Access::kLanes>;
        }
    }
    if (lds > 1 << 16) {
        const hipError_t status = hipFuncSetAttribute(
            reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize,
            static_cast<int>(lds));
        if (status != hipSuccess) {
            return fail(RLN_ERR_HIP, "gated backward_kernel: %s", hipGetErrorString(status));
        }
    }
    const int64_t blocks = a.units < kMaxBlocks ? a.units : kMaxBlocks;
    return launch(kernel, a, blocks, shape.threads, lds, stream, "gated backward_kernel");
}

template <typename X, typename B, int V, bool kPost>
int run(const BackwardArgs& a, const Shape& shape, hipStream_t stream) {
    return a.gate.data != nullptr && a.gate.rows == 1
        ? run_token<X, B, V, kPost, true>(a, shape, stream)
        : run_token<X, B, V, kPost, false>(a, shape, stream);
}
using Args = BackwardArgs;
#endif

template <typename X, typename B, bool kPost>
int slots(const Args& a, const Shape& shape, hipStream_t stream) {
    switch (shape.slots) {
        case 1:
            return run<X, B, 1, kPost>(a, shape, stream);
        case 2:
            return run<X, B, 2, kPost>(a, shape, stream);
        default:
#if RMS_PASS == 1
            if constexpr (kColumns<X> == 8 && kPost) {
                return run<X, B, 3, kPost>(a, shape, stream);
            }
#endif
            if constexpr (kColumns<X> == 4) {
                return run<X, B, 4, kPost>(a, shape, stream);
            }
            return fail(RLN_ERR_UNSUPPORTED, "gated norm: %d slots", shape.slots);
    }
}

template <typename X, typename B>
int post(const Args& a, const Shape& shape, hipStream_t stream) {
    return a.branch_weight != nullptr ? slots<X, B, true>(a, shape, stream)
                                      : slots<X, B, false>(a, shape, stream);
}

template <typename X>
int branch(const Args& a, const Shape& shape, int branch_dtype, hipStream_t stream) {
    switch (branch_dtype) {
        case RLN_DTYPE_F32:
            return post<X, float>(a, shape, stream);
        case RLN_DTYPE_F16:
            return post<X, half_t>(a, shape, stream);
        default:
            return post<X, bf16_t>(a, shape, stream);
    }
}

}  // namespace

#if RMS_PASS == 1
template <typename X>
int launch_forward(const ForwardArgs& a, const Shape& shape, int branch_dtype,
                   hipStream_t stream) {
    return branch<X>(a, shape, branch_dtype, stream);
}
template int launch_forward<RMS_STREAM>(const ForwardArgs&, const Shape&, int, hipStream_t);
#else
template <typename X>
int launch_backward(const BackwardArgs& a, const Shape& shape, int branch_dtype,
                    hipStream_t stream) {
    return branch<X>(a, shape, branch_dtype, stream);
}
template int launch_backward<RMS_STREAM>(const BackwardArgs&, const Shape&, int, hipStream_t);
#endif

}  // namespace gated
}  // namespace rln
