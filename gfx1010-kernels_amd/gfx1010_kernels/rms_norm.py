"""Root-mean-square norm with the residual's addition, for training and serving.

The reference has no such operator (its norm is LayerNorm,
gfx1010_kernels/normalization.py:149-298); names, ``implementation`` modes,
warnings and errors here follow ``residual_layer_norm``:

* :func:`residual_rms_norm` returns ``(updated, normalized)`` with
  ``updated = x + branch`` and its RMS norm, and supports first-order autograd;
  ``checkpoint_dtype=torch.int8`` keeps what the backward needs in 8 bits;
* :func:`residual_rms_norm_quantized` returns the norm in 8 bits with scales,
  for a consumer that multiplies 8-bit activations;
* :func:`dequantize` widens such values again.

Where ``residual_layer_norm`` asks for contiguous fp32 streams, these take a
stream, branch and weight each in fp32, fp16 or bf16, rows of any length from 1
to 16384 at any row stride, and empty tensors. The statistics are fp32. There is
no dropout: models that norm by the root mean square train without it, and
``F.dropout(branch)`` before the call is the same computation.

The PyTorch decomposition (``implementation="torch"``, and what ``"auto"`` falls
back to with a ``RuntimeWarning``) computes the same formulas in fp32 (fp64 for
fp64 tensors), 8-bit codes and checkpoints included.
"""

from __future__ import annotations

import warnings

import torch

from ._normalization_native import TARGET_ARCHITECTURE, _extension, graph_recorded
from ._ops import dequantize_op, residual_rms_norm_op, residual_rms_norm_quantized_op
from .normalization import (
    IMPLEMENTATIONS,
    NO_TANGENTS,
    has_tangent,
    residual_layer_norm_status,
)

MAX_RMS_HIDDEN_SIZE = 16384
STREAM_DTYPES = (torch.float32, torch.float16, torch.bfloat16)
QUANTIZED_DTYPES = (torch.int8, torch.float8_e4m3fn)
GROUP_SIZES = (None, 32, 64, 128, 256)
# Columns under one scale of the 8-bit checkpoint.
CHECKPOINT_GROUP = 128

_STRICT_NATIVE = frozenset({TARGET_ARCHITECTURE, "gfx1010"})
_UNAVAILABLE = f"{TARGET_ARCHITECTURE} native residual RMSNorm is unavailable"
_LARGEST_CODE = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}
_LEAST_MAXIMUM = 2.0 ** -100
# Device indices whose backend status is known to be available.
_READY_DEVICES: set = set()


# The PyTorch decomposition.

def _group_maximum(values, group):
    """max(|values|, 2^-100) over each group of columns, the last one shorter."""
    missing = -values.shape[-1] % group
    if missing:
        values = torch.cat([values, values.new_zeros(*values.shape[:-1], missing)], -1)
    largest = values.unflatten(-1, (-1, group)).abs().amax(-1)
    return torch.where(largest.isnan(), largest, largest.clamp(min=_LEAST_MAXIMUM))


def _codes(values, group, dtype):
    """8-bit codes of fp32 values, and the value of one step per group. A group
    that holds an infinity or a NaN gets NaN for its step."""
    largest = _group_maximum(values, group)
    top = torch.full_like(largest, _LARGEST_CODE[dtype])
    finite = largest.isfinite()
    inverse = torch.where(finite, top / largest, 0.0).repeat_interleave(group, -1)
    steps = (values * inverse[..., :values.shape[-1]]).clamp(-_LARGEST_CODE[dtype],
                                                             _LARGEST_CODE[dtype])
    steps = steps.nan_to_num(nan=0.0)
    codes = (steps.round() if dtype == torch.int8 else steps.float()).to(dtype)
    return codes, torch.where(finite, largest / top, torch.nan)


def _widened(codes, step, group):
    return codes.float() * step.repeat_interleave(group, -1)[..., :codes.shape[-1]]


def _wide(tensor):
    """fp32, or fp64 for an fp64 tensor (which only this path serves)."""
    return tensor if tensor.dtype == torch.float64 else tensor.float()


def _torch_update(x, branch):
    return x if branch is None else (_wide(x) + _wide(branch)).to(x.dtype)


def _rstd(values, eps):
    return 1.0 / torch.sqrt(values.square().mean(-1, keepdim=True) + eps)


class _TorchCheckpointNorm(torch.autograd.Function):
    """The norm of a stream kept for the backward as 8-bit codes."""

    @staticmethod
    def forward(ctx, updated, weight, eps, dtype):
        values = _wide(updated)
        rstd = _rstd(values, eps)
        codes, step = _codes(values, CHECKPOINT_GROUP, torch.int8)
        ctx.save_for_backward(codes, step, rstd, weight)
        ctx.dtype = updated.dtype
        return (values * rstd * _wide(weight)).to(dtype)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_normalized):
        codes, step, rstd, weight = ctx.saved_tensors
        unit = _widened(codes, step, CHECKPOINT_GROUP) * rstd
        upstream = _wide(grad_normalized)
        product = upstream * _wide(weight)
        shared = (product * unit).mean(-1, keepdim=True)
        grad_weight = (upstream * unit).flatten(0, -2).sum(0) if unit.ndim > 1 else upstream * unit
        return ((rstd * (product - unit * shared)).to(ctx.dtype), grad_weight.to(weight.dtype),
                None, None)


def _torch_residual_rms_norm(x, branch, weight, eps, normalized_dtype, checkpoint):
    updated = _torch_update(x, branch)
    dtype = normalized_dtype or x.dtype
    if checkpoint:
        return updated, _TorchCheckpointNorm.apply(updated, weight, eps, dtype)
    values = _wide(updated)
    return updated, (values * _rstd(values, eps) * _wide(weight)).to(dtype)


def _torch_quantized(x, branch, weight, eps, dtype, group_size):
    updated = _torch_update(x, branch)
    values = _wide(updated)
    group = group_size or max(1, values.shape[-1])
    codes, step = _codes(values * _wide(weight), group, dtype)
    return updated, codes, (step * _rstd(values, eps)).float()


def _torch_dequantize(quantized, scale, group_size, dtype):
    return _widened(quantized, scale, group_size or max(1, quantized.shape[-1])).to(dtype)


# Checks and dispatch.

def _input_reason(x, branch, weight, eps):
    """Why the native kernels cannot serve these inputs, or None if they can."""
    tensors = [tensor for tensor in (x, branch, weight) if tensor is not None]
    if not all(tensor.is_cuda for tensor in tensors):
        return "x, branch and weight must be HIP tensors"
    if any(tensor.device != x.device for tensor in tensors):
        return "x, branch and weight must be on the same device"
    if x.ndim < 1 or (branch is not None and branch.shape != x.shape):
        return "x and branch must have the same shape with at least one dimension"
    if not 1 <= x.shape[-1] <= MAX_RMS_HIDDEN_SIZE:
        return f"hidden size must be between 1 and {MAX_RMS_HIDDEN_SIZE}"
    if weight.shape != (x.shape[-1],):
        return "weight must match the final tensor dimension"
    if any(tensor.dtype not in STREAM_DTYPES for tensor in tensors):
        return "x, branch and weight must use float16, bfloat16 or float32"
    if not eps >= 0.0:
        return "eps must not be negative"
    if has_tangent(*tensors):
        return NO_TANGENTS
    return None


def _traced_inputs_served(x, branch, weight, eps):
    """Whether _input_reason finds none. From the extension's check while
    torch.jit.trace runs, which hands out sizes that are tensors of its graph."""
    if torch.jit.is_tracing():
        return _extension()[0].rms_inputs_supported(x, branch, weight, float(eps))
    return _input_reason(x, branch, weight, eps) is None


def _check_implementation(implementation, what="residual RMSNorm"):
    if implementation not in IMPLEMENTATIONS:
        raise ValueError(
            "implementation must be 'auto', 'gfx950', 'gfx1010', 'triton' or 'torch'")
    if implementation == "triton":
        raise RuntimeError(
            f"{TARGET_ARCHITECTURE} {what} is unavailable: "
            "the Triton backend is not part of the MI355X build")


def _native_or_reason(tensor, reason_of, implementation, what="residual RMSNorm"):
    """The native extension, or None and why ``"auto"`` falls back (the answer of
    ``reason_of()``, which the strict modes do not ask); the strict modes and a
    broken install on the target hardware raise."""
    strict = implementation in _STRICT_NATIVE
    unavailable = f"{TARGET_ARCHITECTURE} native {what} is unavailable"
    reason = None if strict else reason_of()
    if strict and not tensor.is_cuda:
        raise RuntimeError(f"{unavailable}: the inputs must be HIP tensors")
    if reason is None:
        if tensor.get_device() not in _READY_DEVICES:
            status = residual_layer_norm_status(tensor.device)
            if not status.available:
                if strict or status.architecture == TARGET_ARCHITECTURE:
                    raise RuntimeError(f"{unavailable}: {status.reason}")
                return None, status.reason
            _READY_DEVICES.add(tensor.get_device())
        # What the strict modes cannot serve raises in the extension.
        return _extension()[0], None
    return None, reason


def _warn(reason, what="residual RMSNorm"):
    warnings.warn(
        f"{TARGET_ARCHITECTURE} native {what} was not used: {reason}",
        RuntimeWarning,
        stacklevel=3,
    )


def residual_rms_norm(
    x,
    branch,
    weight,
    eps=1e-6,
    *,
    implementation="auto",
    normalized_dtype=None,
    checkpoint_dtype=None,
):
    """Fused ``x + branch -> RMS norm``; returns ``(updated, normalized)``.

    ``updated`` is the new residual stream (added in fp32, rounded to ``x``'s
    type) and ``normalized`` is ``updated * rsqrt(mean(updated^2) + eps) *
    weight`` over the last dimension, in ``x``'s type or ``normalized_dtype``.
    ``branch`` has ``x``'s shape, or is None for a norm without an addition;
    ``updated`` is then ``x`` itself. ``x``, ``branch`` and ``weight`` each use
    fp32, fp16 or bf16; tensors whose rows are evenly spaced are read in place,
    others are copied first.

    Supports first-order autograd, HIP graph capture, ``torch.compile``,
    ``torch.jit.trace`` and ``make_fx`` (whose graphs hold the operators
    ``torch.ops.gfx1010_kernels`` registers). Inputs with a forward-mode tangent
    take the PyTorch path, which carries it (the native modes raise, and so does
    ``checkpoint_dtype``, whose norm has no forward-mode derivative). The
    weight's gradient is summed in a fixed order (bitwise reproducible with and
    without ``torch.use_deterministic_algorithms``). The gradients of ``x`` and
    of a branch of the same type are one tensor, as those of ``x + branch`` are.
    With ``checkpoint_dtype=torch.int8`` the backward reads ``updated`` from
    8-bit codes (one fp32 scale for each 128 columns, an error of at most
    1/254 of the group's largest magnitude; the outputs and the norm's statistics
    are not affected) instead of ``updated`` itself, which the graph then no
    longer keeps alive: 1.03 bytes per element instead of 2 or 4.
    """
    _check_implementation(implementation)
    if normalized_dtype is not None and normalized_dtype not in STREAM_DTYPES:
        raise ValueError("normalized_dtype must be None, torch.float32, torch.float16 "
                         "or torch.bfloat16")
    if checkpoint_dtype is not None and checkpoint_dtype != torch.int8:
        raise ValueError("checkpoint_dtype must be None or torch.int8")
    args = (x, branch, weight, eps, normalized_dtype, checkpoint_dtype is not None)
    if implementation == "torch":
        return _torch_residual_rms_norm(*args)
    if torch.compiler.is_compiling():
        reason = _input_reason(x, branch, weight, eps)
        if implementation in _STRICT_NATIVE and reason == NO_TANGENTS:
            raise RuntimeError(f"{_UNAVAILABLE}: {reason}")
        if implementation in _STRICT_NATIVE or reason is None:
            return residual_rms_norm_op(*args)
        return _torch_residual_rms_norm(*args)
    # Inputs the kernels serve, on a device known to be ready: one C++ check and
    # call. The reasons below are only worked out when it declines.
    if implementation == "auto" and x.is_cuda and x.get_device() in _READY_DEVICES:
        result = _extension()[0].residual_rms_norm_if_supported(
            x, branch, weight, float(eps), normalized_dtype, checkpoint_dtype is not None)
        if result is not None:
            return result
    if x.is_cuda and graph_recorded():
        if implementation in _STRICT_NATIVE or _traced_inputs_served(x, branch, weight, eps):
            return residual_rms_norm_op(*args)
        return _torch_residual_rms_norm(*args)
    native, reason = _native_or_reason(
        x, lambda: _input_reason(x, branch, weight, eps), implementation)
    if native is None:
        _warn(reason)
        return _torch_residual_rms_norm(*args)
    return native.residual_rms_norm(x, branch, weight, float(eps), normalized_dtype,
                                    checkpoint_dtype is not None)


def can_use_residual_rms_norm(x, branch, weight, eps=1e-6):
    """True when ``implementation="auto"`` runs natively."""
    return (_input_reason(x, branch, weight, eps) is None
            and residual_layer_norm_status(x.device).available)


def _check_group_size(group_size):
    if group_size not in GROUP_SIZES:
        raise ValueError("group_size must be None, 32, 64, 128 or 256")


def residual_rms_norm_quantized(
    x,
    branch,
    weight,
    eps=1e-6,
    *,
    implementation="auto",
    dtype=torch.float8_e4m3fn,
    group_size=None,
):
    """:func:`residual_rms_norm` with its output in 8 bits; returns
    ``(updated, quantized, scale)``.

    ``quantized`` has ``x``'s shape in ``torch.int8`` (-127 to 127) or
    ``torch.float8_e4m3fn`` (-448 to 448), ``scale`` one fp32 value for each
    token (``[..., 1]``) or, with ``group_size`` 32, 64, 128 or 256, for each
    group of columns (``[..., ceil(hidden / group_size)]``, the last group
    shorter where it does not divide the row): ``quantized * scale`` is the norm,
    each group stepped against its own largest magnitude. A group that holds an
    infinity or a NaN has NaN for its scale.

    For serving: it records no gradient, and raises where one would be lost
    (grad mode on and an input that requires grad, or an input with a
    forward-mode tangent).
    """
    if (implementation == "auto" and x.is_cuda and dtype in QUANTIZED_DTYPES
            and group_size in GROUP_SIZES and x.get_device() in _READY_DEVICES
            and not torch.compiler.is_compiling()):
        result = _extension()[0].residual_rms_norm_quantized_if_supported(
            x, branch, weight, float(eps), dtype, group_size or 0)
        if result is not None:
            return result
    _check_implementation(implementation)
    if dtype not in QUANTIZED_DTYPES:
        raise ValueError("dtype must be torch.int8 or torch.float8_e4m3fn")
    _check_group_size(group_size)
    if torch.is_grad_enabled() and any(
            tensor is not None and tensor.requires_grad for tensor in (x, branch, weight)):
        raise RuntimeError("residual_rms_norm_quantized records no gradient: call it under "
                           "torch.no_grad(), or use residual_rms_norm")
    if has_tangent(x, branch, weight):
        raise RuntimeError("residual_rms_norm_quantized has no forward-mode derivative: call it "
                           "on tensors without a tangent, or use residual_rms_norm")
    args = (x, branch, weight, eps, dtype, group_size)
    if implementation == "torch":
        return _torch_quantized(*args)
    if torch.compiler.is_compiling():
        if implementation in _STRICT_NATIVE or _input_reason(x, branch, weight, eps) is None:
            return residual_rms_norm_quantized_op(*args)
        return _torch_quantized(*args)
    if x.is_cuda and graph_recorded():
        if implementation in _STRICT_NATIVE or _traced_inputs_served(x, branch, weight, eps):
            return residual_rms_norm_quantized_op(*args)
        return _torch_quantized(*args)
    native, reason = _native_or_reason(
        x, lambda: _input_reason(x, branch, weight, eps), implementation)
    if native is None:
        _warn(reason)
        return _torch_quantized(*args)
    return native.residual_rms_norm_quantized(x, branch, weight, float(eps), dtype,
                                              group_size or 0)


def _dequantize_reason(quantized, scale):
    if not quantized.is_cuda or not scale.is_cuda:
        return "quantized and scale must be HIP tensors"
    if quantized.device != scale.device:
        return "quantized and scale must be on the same device"
    return None


def dequantize(quantized, scale, *, group_size=None, dtype=torch.bfloat16,
               implementation="auto"):
    """``quantized * scale`` in ``dtype`` (fp32, fp16 or bf16), for a consumer of
    :func:`residual_rms_norm_quantized`'s output that does not read 8 bits.
    ``group_size`` is the one the values were made with. Records no gradient."""
    if (implementation == "auto" and quantized.is_cuda and dtype in STREAM_DTYPES
            and group_size in GROUP_SIZES and quantized.get_device() in _READY_DEVICES
            and not torch.compiler.is_compiling()):
        result = _extension()[0].dequantize_if_supported(quantized, scale, group_size or 0, dtype)
        if result is not None:
            return result
    _check_implementation(implementation)
    _check_group_size(group_size)
    if dtype not in STREAM_DTYPES:
        raise ValueError("dtype must be torch.float32, torch.float16 or torch.bfloat16")
    if quantized.dtype not in QUANTIZED_DTYPES:
        raise ValueError("quantized must use torch.int8 or torch.float8_e4m3fn")
    if scale.dtype != torch.float32:
        raise ValueError("scale must use torch.float32")
    if quantized.ndim < 1 or quantized.shape[-1] < 1:
        raise ValueError("quantized must have at least one column")
    groups = 1 if group_size is None else -(-quantized.shape[-1] // group_size)
    if tuple(scale.shape) != (*quantized.shape[:-1], groups):
        raise ValueError(f"scale must have shape {(*quantized.shape[:-1], groups)}, one value "
                         "for each group of columns")
    if torch.is_grad_enabled() and scale.requires_grad:
        raise RuntimeError("dequantize records no gradient: call it under torch.no_grad()")
    if has_tangent(quantized, scale):
        raise RuntimeError("dequantize has no forward-mode derivative: call it on tensors without "
                           "a tangent")
    args = (quantized, scale, group_size, dtype)
    if implementation == "torch":
        return _torch_dequantize(*args)
    if torch.compiler.is_compiling():
        if implementation in _STRICT_NATIVE or _dequantize_reason(quantized, scale) is None:
            return dequantize_op(*args)
        return _torch_dequantize(*args)
    if quantized.is_cuda and graph_recorded():
        if implementation in _STRICT_NATIVE or _dequantize_reason(quantized, scale) is None:
            return dequantize_op(*args)
        return _torch_dequantize(*args)
    native, reason = _native_or_reason(
        quantized, lambda: _dequantize_reason(quantized, scale), implementation)
    if native is None:
        _warn(reason)
        return _torch_dequantize(*args)
    return native.dequantize(quantized, scale, group_size or 0, dtype)


__all__ = [
    "can_use_residual_rms_norm",
    "dequantize",
    "residual_rms_norm",
    "residual_rms_norm_quantized",
]
