// Instances of the root-mean-square norm kernels (rms_device.h), one
// translation unit per stream type (RMS_STREAM: float, half_t or bf16_t) and
// pass (RMS_PASS: 1 forward, 2 backward).

#include "rms_device.h"

namespace rln {
namespace rms {
namespace {

template <typename Kernel, typename Args>
int launch(Kernel kernel, const Args& a, int64_t blocks, int threads, size_t lds,
           hipStream_t stream, const char* what) {
    kernel<<<dim3(static_cast<unsigned>(blocks)), threads, lds, stream>>>(a);
    return check_launch(what);
}

#if RMS_PASS == 1
template <typename X, typename B, int V, Mode kMode>
int forward_access(const ForwardArgs& a, const Shape& shape, hipStream_t stream) {
    const int64_t blocks = forward_blocks(a.rows, shape);
    auto kernel = a.words ? forward_kernel<X, B, V, kMode, Access::kWords>
                          : forward_kernel<X, B, V, kMode, Access::kElements>;
    if constexpr (V == 1) {
        if (shape.row_lanes < kWave) {
            kernel = forward_kernel<X, B, 1, kMode, Access::kLanes>;
        }
    }
    return launch(kernel, a, blocks, shape.threads, 0, stream, "rms forward_kernel");
}

template <typename X, typename B, Mode kMode>
int forward_slots(const ForwardArgs& a, const Shape& shape, hipStream_t stream) {
    switch (shape.slots) {
        case 1:
            return forward_access<X, B, 1, kMode>(a, shape, stream);
        case 2:
            return forward_access<X, B, 2, kMode>(a, shape, stream);
        default:
            if constexpr (kColumns<X> == 4) {
                return forward_access<X, B, 4, kMode>(a, shape, stream);
            }
            return fail(RLN_ERR_UNSUPPORTED, "rms forward: %d slots", shape.slots);
    }
}

template <typename X, Mode kMode>
int forward_branch(const ForwardArgs& a, const Shape& shape, int branch_dtype,
                   hipStream_t stream) {
    if (a.branch == nullptr) {
        return forward_slots<X, NoBranch, kMode>(a, shape, stream);
    }
    switch (branch_dtype) {
        case RLN_DTYPE_F32:
            return forward_slots<X, float, kMode>(a, shape, stream);
        case RLN_DTYPE_F16:
            return forward_slots<X, half_t, kMode>(a, shape, stream);
        default:
            return forward_slots<X, bf16_t, kMode>(a, shape, stream);
    }
}
#else
template <typename X, typename Y, int V, bool Checkpoint>
int backward_access(const BackwardArgs& a, const Shape& shape, hipStream_t stream) {
    if (a.slabs > 0) {
        auto kernel = a.words ? backward_kernel<X, Y, V, Checkpoint, Access::kWords, true>
                              : backward_kernel<X, Y, V, Checkpoint, Access::kElements, true>;
        if constexpr (V == 1) {
            if (shape.row_lanes < kWave) {
                kernel = backward_kernel<X, Y, 1, Checkpoint, Access::kLanes, true>;
            }
        }
        return launch(kernel, a, a.slabs + blocks_of(a.rows, shape), shape.threads, 0, stream,
                      "rms backward_kernel");
    }
    const int64_t blocks = backward_blocks(a.rows, shape);
    const size_t lds = a.partials == nullptr
        ? 0 : static_cast<size_t>(teams_of(shape) - 1) * a.hidden * sizeof(float);
    auto kernel = a.words ? backward_kernel<X, Y, V, Checkpoint, Access::kWords, false>
                          : backward_kernel<X, Y, V, Checkpoint, Access::kElements, false>;
    if constexpr (V == 1) {
        if (shape.row_lanes < kWave) {
            kernel = backward_kernel<X, Y, 1, Checkpoint, Access::kLanes, false>;
        }
    }
    return launch(kernel, a, blocks, shape.threads, lds, stream, "rms backward_kernel");
}

template <typename X, typename Y, bool Checkpoint>
int backward_slots(const BackwardArgs& a, const Shape& shape, hipStream_t stream) {
    switch (shape.slots) {
        case 1:
            return backward_access<X, Y, 1, Checkpoint>(a, shape, stream);
        case 2:
            return backward_access<X, Y, 2, Checkpoint>(a, shape, stream);
        default:
            if constexpr (kColumns<X> == 4) {
                return backward_access<X, Y, 4, Checkpoint>(a, shape, stream);
            }
            return fail(RLN_ERR_UNSUPPORTED, "rms backward: %d slots", shape.slots);
    }
}

template <typename X, typename Y>
int backward_kept(const BackwardArgs& a, const Shape& shape, hipStream_t stream) {
    return a.checkpoint != nullptr ? backward_slots<X, Y, true>(a, shape, stream)
                                   : backward_slots<X, Y, false>(a, shape, stream);
}
#endif

}  // namespace

#if RMS_PASS == 1
template <typename X>
int launch_forward(const ForwardArgs& a, const Shape& shape, int branch_dtype, Mode mode,
                   hipStream_t stream) {
    switch (mode) {
        case Mode::kNormalize:
            return forward_branch<X, Mode::kNormalize>(a, shape, branch_dtype, stream);
        case Mode::kCheckpoint:
            return forward_branch<X, Mode::kCheckpoint>(a, shape, branch_dtype, stream);
        default:
            return forward_branch<X, Mode::kQuantize>(a, shape, branch_dtype, stream);
    }
}

template int launch_forward<RMS_STREAM>(const ForwardArgs&, const Shape&, int, Mode, hipStream_t);
#else
template <typename X>
int launch_backward(const BackwardArgs& a, const Shape& shape, int grad_dtype,
                    hipStream_t stream) {
    switch (grad_dtype) {
        case RLN_DTYPE_F32:
            return backward_kept<X, float>(a, shape, stream);
        case RLN_DTYPE_F16:
            return backward_kept<X, half_t>(a, shape, stream);
        default:
            return backward_kept<X, bf16_t>(a, shape, stream);
    }
}

template int launch_backward<RMS_STREAM>(const BackwardArgs&, const Shape&, int, hipStream_t);
#endif

}  // namespace rms
}  // namespace rln
