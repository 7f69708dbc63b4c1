"""``torch.library`` registration of the native residual LayerNorm.

The eager path runs the C++ autograd function of the ``_C`` module
(``_C.residual_layer_norm``, mirroring csrc/residual_layer_norm_bindings.cpp:10-125).
That function is opaque to ``torch.compile``; the two operators registered here
expose the same kernels as functional custom ops with fake (meta) kernels for
shape inference and an autograd formula, so that a compiled graph keeps the
fused op instead of breaking around it (the reference does not support
``torch.compile``; docs/residual_layer_norm.md:301-302).

* ``gfx1010_kernels::rln_forward(x, branch, weight, bias, dropout_p, eps, training,
  normalized_dtype, nonce) -> (updated, normalized, mean, rstd, mask)`` runs
  ``_C.residual_layer_norm_forward`` with the eager path's ``threads``; with
  dropout it reserves its Philox offsets from the device's default generator
  when it executes, exactly as the eager path does, so compiled and eager runs
  draw the same masks from the same RNG state. ``nonce`` is a fresh zero-size
  tensor per call (``residual_layer_norm_op`` makes it): the op draws from the
  generator, so two calls with equal arguments are different computations,
  and the nonce keeps a compiler from merging them. AOTAutograd's common
  subexpression pass merges identical calls of a functional custom op, but
  never two ``aten.empty`` nodes, so each call's nonce differs.
* ``gfx1010_kernels::rln_backward(grad_updated, grad_normalized, updated, weight,
  mean, rstd, mask, dropout_p, training, branch_dtype, compute_parameters)
  -> (grad_x, grad_branch, grad_weight, grad_bias)`` runs
  ``_C.residual_layer_norm_backward``; a missing upstream gradient counts as
  zero, and the weight/bias gradients are zero when ``grad_normalized`` is.
  With ``compute_parameters`` false (the backward pass needs neither weight
  nor bias gradient: frozen parameters, or gradients taken for the inputs
  only) the weight/bias sums are skipped and those two outputs are empty.
* ``gfx1010_kernels::rms_forward`` / ``rms_backward`` / ``rms_quantized`` /
  ``dequantize`` do the same for the root-mean-square norm
  (``_C.residual_rms_norm_*``). They draw nothing, so equal calls may be merged.
* ``gfx1010_kernels::gated_forward`` / ``gated_backward`` and ``rotary_forward`` /
  ``rotary_backward`` do so for the gated residual norm and the rotary norm of heads
  (``_C.gated_residual_rms_norm_*``, ``_C.rms_norm_rotary_*``); ``needed`` has bit ``i``
  set where the gradient of tensor input ``i`` is asked for, and an output that is
  not asked for, or does not exist, is empty.

``torch.jit.trace`` and ``make_fx`` record these operators as well.
"""

from __future__ import annotations

from typing import Optional, Sequence

import torch
from torch import Tensor

from ._normalization_native import TARGET_ARCHITECTURE, _extension, launch_threads

_NAMESPACE = "gfx1010_kernels"

# Interface-compatibility launch hints the raw backward range-checks
# (threads, block_rows, parameter_threads, parameter_groups).
_BACKWARD_HINTS = (128, 64, 64, 1)


def _native():
    extension, reason = _extension()
    if extension is None:
        raise RuntimeError(f"{TARGET_ARCHITECTURE} native extension is unavailable: {reason}")
    return extension


@torch.library.custom_op(f"{_NAMESPACE}::rln_forward", mutates_args=(), device_types="cuda")
def rln_forward(
    x: Tensor,
    branch: Tensor,
    weight: Tensor,
    bias: Tensor,
    dropout_p: float,
    eps: float,
    training: bool,
    normalized_dtype: Optional[torch.dtype] = None,
    nonce: Optional[Tensor] = None,
) -> tuple[Tensor, Tensor, Tensor, Tensor, Tensor]:
    return tuple(
        _native().residual_layer_norm_forward(
            x, branch, weight, bias, float(dropout_p), float(eps), bool(training),
            launch_threads(x.shape[-1]),
            normalized_dtype=normalized_dtype,
        )
    )


@rln_forward.register_fake
def _rln_forward_fake(x, branch, weight, bias, dropout_p, eps, training, normalized_dtype=None,
                      nonce=None):
    hidden = x.shape[-1]
    rows = x.numel() // hidden
    mask_words = rows * (hidden // 32) if (training and dropout_p > 0.0) else 0
    return (
        torch.empty_like(x, memory_format=torch.contiguous_format),
        torch.empty_like(x, dtype=normalized_dtype or torch.float32,
                         memory_format=torch.contiguous_format),
        x.new_empty((rows,)),
        x.new_empty((rows,)),
        x.new_empty((mask_words,), dtype=torch.int32),
    )


@torch.library.custom_op(f"{_NAMESPACE}::rln_backward", mutates_args=(), device_types="cuda")
def rln_backward(
    grad_updated: Optional[Tensor],
    grad_normalized: Optional[Tensor],
    updated: Tensor,
    weight: Tensor,
    mean: Tensor,
    rstd: Tensor,
    mask: Tensor,
    dropout_p: float,
    training: bool,
    branch_dtype: torch.dtype,
    compute_parameters: bool = True,
) -> tuple[Tensor, Tensor, Tensor, Tensor]:
    grad_x, grad_branch, grad_weight, grad_bias = _native().residual_layer_norm_backward(
        grad_updated, grad_normalized, updated, weight, mean, rstd, mask, float(dropout_p),
        bool(training), branch_dtype == torch.float16, *_BACKWARD_HINTS,
        bool(compute_parameters), branch_dtype=branch_dtype,
    )
    if not compute_parameters:
        grad_weight = updated.new_empty((0,))
        grad_bias = updated.new_empty((0,))
    return grad_x, grad_branch, grad_weight, grad_bias


@rln_backward.register_fake
def _rln_backward_fake(grad_updated, grad_normalized, updated, weight, mean, rstd, mask,
                       dropout_p, training, branch_dtype, compute_parameters=True):
    hidden = updated.shape[-1] if compute_parameters else 0
    return (
        torch.empty_like(updated, memory_format=torch.contiguous_format),
        torch.empty_like(updated, dtype=branch_dtype, memory_format=torch.contiguous_format),
        updated.new_empty((hidden,)),
        updated.new_empty((hidden,)),
    )


def _setup_context(ctx, inputs, output):
    _, branch, weight, _, dropout_p, _, training, _, _ = inputs
    updated, _, mean, rstd, mask = output
    ctx.save_for_backward(updated, weight, mean, rstd, mask)
    ctx.dropout_p = dropout_p
    ctx.training = training
    ctx.branch_dtype = branch.dtype
    ctx.mark_non_differentiable(mean, rstd, mask)
    ctx.set_materialize_grads(False)


def _backward(ctx, grad_updated, grad_normalized, _grad_mean, _grad_rstd, _grad_mask):
    if grad_updated is None and grad_normalized is None:
        return None, None, None, None, None, None, None, None, None
    updated, weight, mean, rstd, mask = ctx.saved_tensors
    if grad_updated is not None:
        grad_updated = grad_updated.contiguous()
    if grad_normalized is not None:
        grad_normalized = grad_normalized.contiguous()
    # Weight/bias sums only when this backward pass asks for them.
    parameters = grad_normalized is not None and (ctx.needs_input_grad[2]
                                                  or ctx.needs_input_grad[3])
    grad_x, grad_branch, grad_weight, grad_bias = rln_backward(
        grad_updated, grad_normalized, updated, weight, mean, rstd, mask, ctx.dropout_p,
        ctx.training, ctx.branch_dtype, parameters,
    )
    if not parameters:
        grad_weight = grad_bias = None
    return grad_x, grad_branch, grad_weight, grad_bias, None, None, None, None, None


rln_forward.register_autograd(_backward, setup_context=_setup_context)


def residual_layer_norm_op(x, branch, weight, bias, dropout_p, eps, training,
                           normalized_dtype=None):
    """``(updated, normalized)`` through the registered custom op. Each call
    passes a new zero-size nonce, so two dropout calls on equal arguments stay
    two draws under ``torch.compile``."""
    nonce = torch.empty(0, device=x.device)
    updated, normalized, _, _, _ = rln_forward(
        x, branch, weight, bias, float(dropout_p), float(eps), bool(training), normalized_dtype,
        nonce,
    )
    return updated, normalized


@torch.library.custom_op(f"{_NAMESPACE}::rms_forward", mutates_args=(), device_types="cuda")
def rms_forward(
    x: Tensor,
    branch: Optional[Tensor],
    weight: Tensor,
    eps: float,
    normalized_dtype: Optional[torch.dtype] = None,
    checkpoint: bool = False,
) -> tuple[Tensor, Tensor, Tensor]:
    return _native().residual_rms_norm_forward(x, branch, weight, float(eps), normalized_dtype,
                                               checkpoint)


def _rms_state_bytes(rows, hidden, checkpoint):
    """Bytes of the state tensor (rstd; with the checkpoint its scales and
    codes), as rms_torch.cpp lays it out."""
    if not checkpoint:
        return 4 * rows
    groups = (hidden + 127) // 128
    return (4 * rows + 255) // 256 * 256 + (4 * rows * groups + 255) // 256 * 256 + rows * hidden


@rms_forward.register_fake
def _rms_forward_fake(x, branch, weight, eps, normalized_dtype=None, checkpoint=False):
    hidden = x.shape[-1]
    rows = x.numel() // hidden
    return (
        x.new_empty((0,)) if branch is None else x.new_empty(x.shape),
        x.new_empty(x.shape, dtype=normalized_dtype or x.dtype),
        x.new_empty((_rms_state_bytes(rows, hidden, checkpoint),), dtype=torch.uint8),
    )


@torch.library.custom_op(f"{_NAMESPACE}::rms_backward", mutates_args=(), device_types="cuda")
def rms_backward(
    grad_updated: Optional[Tensor],
    grad_normalized: Tensor,
    updated: Optional[Tensor],
    state: Tensor,
    weight: Tensor,
    x_dtype: torch.dtype,
    branch_dtype: Optional[torch.dtype],
    checkpoint: bool,
    weight_gradient: bool,
) -> tuple[Tensor, Tensor, Tensor]:
    grad_x, grad_branch, grad_weight = _native().residual_rms_norm_backward(
        grad_updated, grad_normalized, updated, state, weight, x_dtype, branch_dtype, checkpoint,
        weight_gradient)
    empty = grad_x.new_empty((0,))
    return (grad_x, empty if grad_branch is None else grad_branch,
            empty.clone() if grad_weight is None else grad_weight)


@rms_backward.register_fake
def _rms_backward_fake(grad_updated, grad_normalized, updated, state, weight, x_dtype,
                       branch_dtype, checkpoint, weight_gradient):
    own_branch = branch_dtype is not None and branch_dtype != x_dtype
    return (
        grad_normalized.new_empty(grad_normalized.shape, dtype=x_dtype),
        grad_normalized.new_empty(grad_normalized.shape, dtype=branch_dtype) if own_branch
        else grad_normalized.new_empty((0,), dtype=x_dtype),
        weight.new_empty(weight.shape) if weight_gradient
        else grad_normalized.new_empty((0,), dtype=x_dtype),
    )


def _rms_setup_context(ctx, inputs, output):
    x, branch, weight, _, _, checkpoint = inputs
    updated, _, state = output
    kept = None if checkpoint else x if branch is None else updated
    ctx.save_for_backward(kept, weight, state)
    ctx.x_dtype = x.dtype
    ctx.branch_dtype = None if branch is None else branch.dtype
    ctx.checkpoint = checkpoint
    ctx.mark_non_differentiable(*([updated, state] if branch is None else [state]))
    ctx.set_materialize_grads(False)


def _rms_backward_formula(ctx, grad_updated, grad_normalized, _grad_state):
    grads = [None] * 6
    if grad_normalized is None:
        if grad_updated is not None:
            grads[0] = grad_updated
            grads[1] = grad_updated.to(ctx.branch_dtype)
        return tuple(grads)
    kept, weight, state = ctx.saved_tensors
    grad_x, grad_branch, grad_weight = rms_backward(
        grad_updated if ctx.branch_dtype is not None else None, grad_normalized, kept, state,
        weight, ctx.x_dtype, ctx.branch_dtype, ctx.checkpoint, ctx.needs_input_grad[2])
    grads[0] = grad_x
    if ctx.branch_dtype is not None:
        grads[1] = grad_x if ctx.branch_dtype == ctx.x_dtype else grad_branch
    if ctx.needs_input_grad[2]:
        grads[2] = grad_weight
    return tuple(grads)


rms_forward.register_autograd(_rms_backward_formula, setup_context=_rms_setup_context)


def residual_rms_norm_op(x, branch, weight, eps, normalized_dtype=None, checkpoint=False):
    """``(updated, normalized)`` through the registered custom op. A compiled call that
    records no gradient writes no checkpoint (grad mode and what requires a gradient
    are guarded by the compiler; other recorded graphs may run under any)."""
    if checkpoint and torch.compiler.is_compiling():
        checkpoint = torch.is_grad_enabled() and any(
            tensor is not None and tensor.requires_grad for tensor in (x, branch, weight))
    updated, normalized, _ = rms_forward(x, branch, weight, float(eps), normalized_dtype,
                                         checkpoint)
    return (x if branch is None else updated), normalized


@torch.library.custom_op(f"{_NAMESPACE}::rms_quantized", mutates_args=(), device_types="cuda")
def rms_quantized(
    x: Tensor,
    branch: Optional[Tensor],
    weight: Tensor,
    eps: float,
    dtype: torch.dtype,
    group: int,
) -> tuple[Tensor, Tensor, Tensor]:
    updated, quantized, scale = _native().residual_rms_norm_quantized(
        x, branch, weight, float(eps), dtype, group)
    return (x.new_empty((0,)) if branch is None else updated), quantized, scale


@rms_quantized.register_fake
def _rms_quantized_fake(x, branch, weight, eps, dtype, group):
    groups = 1 if group == 0 else (x.shape[-1] + group - 1) // group
    return (
        x.new_empty((0,)) if branch is None else x.new_empty(x.shape),
        x.new_empty(x.shape, dtype=dtype),
        x.new_empty((*x.shape[:-1], groups), dtype=torch.float32),
    )


def residual_rms_norm_quantized_op(x, branch, weight, eps, dtype, group_size):
    """``(updated, quantized, scale)`` through the registered custom op."""
    updated, quantized, scale = rms_quantized(x, branch, weight, float(eps), dtype,
                                              group_size or 0)
    return (x if branch is None else updated), quantized, scale


@torch.library.custom_op(f"{_NAMESPACE}::dequantize", mutates_args=(), device_types="cuda")
def dequantize(quantized: Tensor, scale: Tensor, group: int, dtype: torch.dtype) -> Tensor:
    return _native().dequantize(quantized, scale, group, dtype)


@dequantize.register_fake
def _dequantize_fake(quantized, scale, group, dtype):
    return quantized.new_empty(quantized.shape, dtype=dtype)


def dequantize_op(quantized, scale, group_size, dtype):
    """The widened values through the registered custom op."""
    return dequantize(quantized, scale, group_size or 0, dtype)


def _or_empty(tensor, like):
    """``tensor``, or an empty one: an operator returns every output."""
    return like.new_empty((0,)) if tensor is None else tensor


@torch.library.custom_op(f"{_NAMESPACE}::gated_forward", mutates_args=(), device_types="cuda")
def gated_forward(
    x: Tensor,
    branch: Tensor,
    weight: Tensor,
    branch_weight: Optional[Tensor],
    gate: Optional[Tensor],
    eps: float,
    branch_eps: float,
    residual_scale: float,
    branch_scale: float,
    normalized_dtype: Optional[torch.dtype] = None,
) -> tuple[Tensor, Tensor, Tensor]:
    return _native().gated_residual_rms_norm_forward(
        x, branch, weight, branch_weight, gate, float(eps), float(branch_eps),
        float(residual_scale), float(branch_scale), normalized_dtype)


@gated_forward.register_fake
def _gated_forward_fake(x, branch, weight, branch_weight, gate, eps, branch_eps, residual_scale,
                        branch_scale, normalized_dtype=None):
    rows = x.numel() // x.shape[-1]
    return (
        x.new_empty(x.shape),
        x.new_empty(x.shape, dtype=normalized_dtype or x.dtype),
        x.new_empty((rows if branch_weight is None else 2 * rows,), dtype=torch.float32),
    )


@torch.library.custom_op(f"{_NAMESPACE}::gated_backward", mutates_args=(), device_types="cuda")
def gated_backward(
    grad_updated: Optional[Tensor],
    grad_normalized: Optional[Tensor],
    updated: Tensor,
    branch: Tensor,
    weight: Tensor,
    branch_weight: Optional[Tensor],
    gate: Optional[Tensor],
    statistics: Tensor,
    residual_scale: float,
    branch_scale: float,
    needed: int,
) -> tuple[Tensor, Tensor, Tensor, Tensor, Tensor]:
    gradients = _native().gated_residual_rms_norm_backward(
        grad_updated, grad_normalized, updated, branch, weight, branch_weight, gate, statistics,
        float(residual_scale), float(branch_scale), needed)
    return tuple(_or_empty(gradient, updated) for gradient in gradients)


@gated_backward.register_fake
def _gated_backward_fake(grad_updated, grad_normalized, updated, branch, weight, branch_weight,
                         gate, statistics, residual_scale, branch_scale, needed):
    def like(tensor, wanted):
        if not wanted or tensor is None:
            return updated.new_empty((0,))
        return tensor.new_empty(tensor.shape)

    return (
        updated.new_empty(updated.shape),
        branch.new_empty(branch.shape),
        like(weight, needed >> 2 & 1 and grad_normalized is not None),
        like(branch_weight, needed >> 3 & 1),
        like(gate, needed >> 4 & 1),
    )


def _needed(flags):
    return sum(1 << index for index, flag in enumerate(flags) if flag)


def _gated_setup_context(ctx, inputs, output):
    _, branch, weight, branch_weight, gate, _, _, ctx.residual_scale, ctx.branch_scale, _ = inputs
    updated, _, statistics = output
    ctx.save_for_backward(updated, branch, weight, branch_weight, gate, statistics)
    ctx.mark_non_differentiable(statistics)
    ctx.set_materialize_grads(False)


def _gated_backward_formula(ctx, grad_updated, grad_normalized, _grad_statistics):
    grads = [None] * 10
    if grad_updated is None and grad_normalized is None:
        return tuple(grads)
    needed = _needed(ctx.needs_input_grad[:5])
    if grad_normalized is None:
        needed &= ~4
    gradients = gated_backward(grad_updated, grad_normalized, *ctx.saved_tensors,
                               ctx.residual_scale, ctx.branch_scale, needed)
    for index in range(5):
        if needed >> index & 1:
            grads[index] = gradients[index]
    return tuple(grads)


gated_forward.register_autograd(_gated_backward_formula, setup_context=_gated_setup_context)


def gated_residual_rms_norm_op(*args):
    """``(updated, normalized)`` through the registered custom op."""
    updated, normalized, _ = gated_forward(*args)
    return updated, normalized


@torch.library.custom_op(f"{_NAMESPACE}::rotary_forward", mutates_args=(), device_types="cuda")
def rotary_forward(
    q: Tensor,
    k: Optional[Tensor],
    positions: Tensor,
    inverse_frequencies: Tensor,
    sections: Sequence[int],
    cyclic: bool,
    interleaved: bool,
    q_weight: Optional[Tensor],
    k_weight: Optional[Tensor],
    eps: float,
) -> tuple[Tensor, Tensor]:
    return _native().rms_norm_rotary_forward(
        q, k, positions, inverse_frequencies, list(sections), cyclic, interleaved, q_weight,
        k_weight, float(eps))


@rotary_forward.register_fake
def _rotary_forward_fake(q, k, positions, inverse_frequencies, sections, cyclic, interleaved,
                         q_weight, k_weight, eps):
    return q.new_empty(q.shape), q.new_empty((0,) if k is None else k.shape)


@torch.library.custom_op(f"{_NAMESPACE}::rotary_backward", mutates_args=(), device_types="cuda")
def rotary_backward(
    grad_q: Optional[Tensor],
    grad_k: Optional[Tensor],
    q: Optional[Tensor],
    k: Optional[Tensor],
    positions: Tensor,
    inverse_frequencies: Tensor,
    sections: Sequence[int],
    cyclic: bool,
    interleaved: bool,
    q_weight: Optional[Tensor],
    k_weight: Optional[Tensor],
    eps: float,
    needed: int,
) -> tuple[Tensor, Tensor, Tensor, Tensor]:
    gradients = _native().rms_norm_rotary_backward(
        grad_q, grad_k, q, k, positions, inverse_frequencies, list(sections), cyclic, interleaved,
        q_weight, k_weight, float(eps), needed)
    like = grad_k if grad_q is None else grad_q
    return tuple(_or_empty(gradient, like) for gradient in gradients)


@rotary_backward.register_fake
def _rotary_backward_fake(grad_q, grad_k, q, k, positions, inverse_frequencies, sections, cyclic,
                          interleaved, q_weight, k_weight, eps, needed):
    base = grad_k if grad_q is None else grad_q

    def like(tensor, wanted=True):
        if tensor is None or not wanted:
            return base.new_empty((0,))
        return tensor.new_empty(tensor.shape)

    return (like(grad_q), like(grad_k),
            like(q_weight, grad_q is not None and needed >> 2 & 1),
            like(k_weight, grad_k is not None and needed >> 3 & 1))


def _rotary_setup_context(ctx, inputs, output):
    # The operator's own kernel runs without grad mode and cannot tell.
    if ctx.needs_input_grad[2] or ctx.needs_input_grad[3]:
        raise RuntimeError("rotary RMSNorm: positions and inverse_frequencies have no gradient")
    (q, k, positions, frequencies, ctx.sections, ctx.cyclic, ctx.interleaved, q_weight, k_weight,
     ctx.eps) = inputs
    ctx.save_for_backward(None if q_weight is None else q, None if k_weight is None else k,
                          positions, frequencies, q_weight, k_weight)
    ctx.has_k = k is not None
    if k is None:
        ctx.mark_non_differentiable(output[1])
    ctx.set_materialize_grads(False)


def _rotary_backward_formula(ctx, grad_q, grad_k):
    grads = [None] * 10
    if not ctx.has_k:
        grad_k = None
    if grad_q is None and grad_k is None:
        return tuple(grads)
    q, k, positions, frequencies, q_weight, k_weight = ctx.saved_tensors
    places = (0, 1, 7, 8)
    needed = _needed(ctx.needs_input_grad[place] for place in places)
    needed &= ~((0 if grad_q is not None else 5) | (0 if grad_k is not None else 10))
    gradients = rotary_backward(grad_q, grad_k, q, k, positions, frequencies, ctx.sections,
                                ctx.cyclic, ctx.interleaved, q_weight, k_weight, ctx.eps, needed)
    for index, place in enumerate(places):
        if needed >> index & 1:
            grads[place] = gradients[index]
    return tuple(grads)


rotary_forward.register_autograd(_rotary_backward_formula, setup_context=_rotary_setup_context)


def rms_norm_rotary_op(q, k, *args):
    """``(q, k)`` through the registered custom op."""
    q_out, k_out = rotary_forward(q, k, *args)
    return q_out, None if k is None else k_out


__all__ = [
    "dequantize",
    "dequantize_op",
    "gated_backward",
    "gated_forward",
    "gated_residual_rms_norm_op",
    "residual_layer_norm_op",
    "residual_rms_norm_op",
    "residual_rms_norm_quantized_op",
    "rln_backward",
    "rln_forward",
    "rms_backward",
    "rms_forward",
    "rms_norm_rotary_op",
    "rms_quantized",
    "rotary_backward",
    "rotary_forward",
]
