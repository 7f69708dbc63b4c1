"""Norms before and after a block, fused with the block's gate and the residual's scale.

The reference has no such operator; names, ``implementation`` modes, warnings
and errors here follow ``residual_rms_norm``. :func:`gated_residual_rms_norm` takes
the output of a block (attention, an MLP), norms it by its root mean square where it
has a weight for that, gates and scales it, adds it to the scaled stream and norms
the sum for the next block:

    a          = RMS norm of branch * branch_weight     (branch itself without one)
    updated    = residual_scale * x + branch_scale * gate * a
    normalized = RMS norm of updated * weight

with first-order autograd for ``x``, ``branch``, ``weight``, ``branch_weight`` and
``gate``. What each factor is made of stays with the caller: a gate ``tanh(g)``, a weight
``w * (1 + scale)`` of a conditioned model or ``1 + w`` are small tensors of their own.
"""

from __future__ import annotations

import math

import torch

from ._normalization_native import TARGET_ARCHITECTURE, _extension, graph_recorded
from ._ops import gated_residual_rms_norm_op
from .normalization import NO_TANGENTS, has_tangent, residual_layer_norm_status
from .rms_norm import (
    MAX_RMS_HIDDEN_SIZE,
    STREAM_DTYPES,
    _check_implementation,
    _native_or_reason,
    _READY_DEVICES,
    _rstd,
    _STRICT_NATIVE,
    _warn,
    _wide,
)

_DTYPES_OR_NONE = (None, *STREAM_DTYPES)
_WHAT = "gated residual RMSNorm"


# The PyTorch decomposition.

def _torch_gated(x, branch, weight, branch_weight, gate, eps, branch_eps, residual_scale,
                 branch_scale, normalized_dtype):
    added = _wide(branch)
    if branch_weight is not None:
        added = added * _rstd(added, branch_eps) * _wide(branch_weight)
    if gate is not None:
        added = added * _wide(gate)
    updated = (residual_scale * _wide(x) + branch_scale * added).to(x.dtype)
    values = _wide(updated)
    normalized = values * _rstd(values, eps) * _wide(weight)
    return updated, normalized.to(normalized_dtype or x.dtype)


# Checks and dispatch.

def _shared_rows(factor, x):
    """The rows of ``x`` that share a row of ``factor``, or 0 where its shape does
    not repeat over whole runs of them."""
    missing = x.ndim - factor.ndim
    if factor.ndim < 1 or missing < 0 or factor.shape[-1] != x.shape[-1]:
        return 0
    sizes = (1,) * missing + tuple(factor.shape)
    rows, index = 1, x.ndim - 2
    while index >= 0 and sizes[index] == 1:
        rows *= x.shape[index]
        index -= 1
    return rows if sizes[:index + 1] == tuple(x.shape[:index + 1]) else 0


def _input_reason(x, branch, weight, branch_weight, gate, eps, branch_eps, residual_scale,
                  branch_scale):
    """Why the native kernels cannot serve these inputs, or None if they can."""
    tensors = [tensor for tensor in (x, branch, weight, branch_weight, gate) if tensor is not None]
    if not all(tensor.is_cuda for tensor in tensors):
        return "all tensors must be HIP tensors"
    if any(tensor.device != x.device for tensor in tensors):
        return "all tensors must be on the same HIP device"
    if any(tensor.dtype not in STREAM_DTYPES for tensor in tensors):
        return "all tensors must use float16, bfloat16 or float32"
    if has_tangent(*tensors):
        return NO_TANGENTS
    if x.ndim < 1 or branch.shape != x.shape:
        return "x and branch must have the same shape with at least one dimension"
    hidden = x.shape[-1]
    if not 1 <= hidden <= MAX_RMS_HIDDEN_SIZE:
        return f"hidden size must be between 1 and {MAX_RMS_HIDDEN_SIZE}"
    if branch_weight is not None and branch_weight.shape != (hidden,):
        return "branch_weight must match the hidden size"
    rows = x.numel() // hidden
    if rows > 0:
        weight_rows = _shared_rows(weight, x)
        gate_rows = rows if gate is None else _shared_rows(gate, x)
        if weight_rows == 0 or gate_rows == 0:
            return "gate and weight must repeat over the last of x's leading dimensions"
        if not (gate_rows <= 1 or gate_rows >= rows or weight_rows >= rows
                or gate_rows == weight_rows):
            return "gate and weight must repeat over the same rows"
    elif any(factor.ndim < 1 or factor.shape[-1] != hidden
             for factor in (weight, gate) if factor is not None):
        return "gate and weight must match the hidden size"
    if not (eps >= 0.0 and branch_eps >= 0.0):
        return "eps must not be negative"
    # By comparisons, which a graph of torch.compile with symbolic numbers can hold.
    if not all(-math.inf < scale < math.inf for scale in (residual_scale, branch_scale)):
        return "residual_scale and branch_scale must be finite"
    return None


def _traced_reason(*args):
    """_input_reason, from the extension's check while torch.jit.trace runs, which
    hands out sizes that are tensors of its graph."""
    if torch.jit.is_tracing():
        return _extension()[0].gated_inputs_refusal(*args)
    return _input_reason(*args)


def check_scales(residual_scale, branch_scale):
    """Scales are numbers; a tensor's gradient would be lost with its conversion."""
    for name, scale in (("residual_scale", residual_scale), ("branch_scale", branch_scale)):
        if isinstance(scale, torch.Tensor) and scale.requires_grad and torch.is_grad_enabled():
            raise ValueError(f"{name} is a number and has no gradient: pass a learned scale of "
                             "the branch as its gate")


def _check_shapes(x, branch, weight, branch_weight, gate):
    """What no implementation takes: tensors that do not fit one another."""
    if x.ndim < 1 or branch.shape != x.shape:
        raise ValueError("x and branch must have the same shape with at least one dimension")
    if branch_weight is not None and branch_weight.shape != x.shape[-1:]:
        raise ValueError("branch_weight must match the final dimension")
    for name, factor in (("weight", weight), ("gate", gate)):
        if factor is None:
            continue
        missing = x.ndim - factor.ndim
        if (factor.ndim < 1 or missing < 0 or factor.shape[-1] != x.shape[-1]
                or any(own not in (1, size) for own, size in zip(factor.shape, x.shape[missing:]))):
            raise ValueError(f"{name} must match the final dimension and broadcast over the others")


def gated_residual_rms_norm(
    x,
    branch,
    weight,
    eps=1e-6,
    *,
    branch_weight=None,
    branch_eps=None,
    gate=None,
    residual_scale=1.0,
    branch_scale=1.0,
    implementation="auto",
    normalized_dtype=None,
):
    """Fused ``residual_scale * x + branch_scale * gate * RMS norm(branch)`` and the RMS
    norm of it; returns ``(updated, normalized)``.

    ``branch`` has ``x``'s shape ``[..., hidden]``. With ``branch_weight`` (``[hidden]``) it
    is normed first, with ``branch_eps`` (None: ``eps``). The scales are numbers; one that
    is learned is a gate. ``gate`` is None, ``[hidden]``, or has ``x``'s leading dimensions
    from the first one on and 1 in the rest (``[batch, 1, hidden]`` for one a sample,
    ``x``'s shape for one a token); ``weight``, of the last norm, may have the same shapes.
    ``updated`` is computed in fp32 and rounded to ``x``'s type, ``normalized`` is the norm
    of the rounded stream in ``x``'s type or ``normalized_dtype``. Every tensor uses fp32,
    fp16 or bf16, each its own; tensors whose rows are evenly spaced are read in place. The
    kernels take 1 to 16384 columns and a gate and a weight that, where both differ between
    samples, differ between the same ones; ``implementation="auto"`` computes other shapes
    that broadcast over ``x`` in PyTorch, with a ``RuntimeWarning``.

    Supports first-order autograd, HIP graph capture, ``torch.compile``,
    ``torch.jit.trace`` and ``make_fx``, as :func:`residual_rms_norm` does; inputs with a
    forward-mode tangent take the PyTorch path. The gradients of ``weight``,
    ``branch_weight`` and ``gate`` are summed in fp32 in a fixed order (bitwise
    reproducible); a weight whose rows serve few tokens each costs several times its bytes
    there. The graph keeps ``updated``, ``branch`` and the factors, and four or eight bytes
    per row.
    """
    if type(residual_scale) is not float or type(branch_scale) is not float:
        check_scales(residual_scale, branch_scale)
    if (implementation == "auto" and x.is_cuda and x.get_device() in _READY_DEVICES
            and normalized_dtype in _DTYPES_OR_NONE and not torch.compiler.is_compiling()):
        result = _extension()[0].gated_residual_rms_norm_if_supported(
            x, branch, weight, branch_weight, gate, float(eps),
            float(eps if branch_eps is None else branch_eps), float(residual_scale),
            float(branch_scale), normalized_dtype)
        if result is not None:
            return result
    _check_implementation(implementation, _WHAT)
    if normalized_dtype not in _DTYPES_OR_NONE:
        raise ValueError("normalized_dtype must be None, torch.float32, torch.float16 "
                         "or torch.bfloat16")
    _check_shapes(x, branch, weight, branch_weight, gate)
    args = (x, branch, weight, branch_weight, gate, float(eps),
            float(eps if branch_eps is None else branch_eps), float(residual_scale),
            float(branch_scale))
    strict = implementation in _STRICT_NATIVE
    if implementation == "torch":
        return _torch_gated(*args, normalized_dtype)
    if torch.compiler.is_compiling():
        reason = _input_reason(*args)
        if strict and reason == NO_TANGENTS:
            raise RuntimeError(f"{TARGET_ARCHITECTURE} native {_WHAT} is unavailable: {reason}")
        if strict or reason is None:
            return gated_residual_rms_norm_op(*args, normalized_dtype)
        return _torch_gated(*args, normalized_dtype)
    if x.is_cuda and graph_recorded():
        if strict or _traced_reason(*args) is None:
            return gated_residual_rms_norm_op(*args, normalized_dtype)
        return _torch_gated(*args, normalized_dtype)
    native, reason = _native_or_reason(x, lambda: _input_reason(*args), implementation, _WHAT)
    if native is None:
        _warn(reason, _WHAT)
        return _torch_gated(*args, normalized_dtype)
    return native.gated_residual_rms_norm(*args, normalized_dtype)


def can_use_gated_residual_rms_norm(x, branch, weight, eps=1e-6, *, branch_weight=None,
                                    branch_eps=None, gate=None, residual_scale=1.0,
                                    branch_scale=1.0):
    """True when ``implementation="auto"`` runs natively."""
    reason = _input_reason(x, branch, weight, branch_weight, gate, float(eps),
                           float(eps if branch_eps is None else branch_eps),
                           float(residual_scale), float(branch_scale))
    return reason is None and residual_layer_norm_status(x.device).available


__all__ = [
    "can_use_gated_residual_rms_norm",
    "gated_residual_rms_norm",
]
