"""Pre-norm transformer integration of the fused residual LayerNorm.

The reference documents the integration as a recipe
(docs/residual_layer_norm.md:51-83): replace ``x = x + branch; h = ln(x)`` by
one ``residual_layer_norm`` call that takes the parameters of the LayerNorm
that *consumes* the new residual stream, pass the sublayer's pre-dropout
output with the original dropout probability, and keep the existing
``LayerNorm`` modules so that checkpoint ``state_dict`` keys do not change.
This module is that recipe as code:

* :func:`residual_norm` fuses one ``x + dropout(branch)`` with the
  ``nn.LayerNorm`` that follows it, reading the module's weight, bias and eps;
* :func:`prenorm_forward` runs a stack of pre-norm blocks
  (``h = ln_1(x); x = x + drop(attn(h)); h = ln_2(x); x = x + drop(mlp(h))``
  per block, then the final norm) with every residual add fused into the
  norm after it: a block's ``ln_2`` after its attention, the next
  block's ``ln_1`` after its MLP, and the final norm after the last MLP. Only
  the first ``ln_1`` (no residual add before it) runs as a plain LayerNorm.

Both take ``nn.RMSNorm`` modules as well, through ``residual_rms_norm``.

Neither function owns parameters: they read the caller's modules, so a model
that switches its ``forward`` to them keeps its ``state_dict`` unchanged.
"""

from __future__ import annotations

from typing import Callable, Sequence, Union

import torch
from torch import nn
from torch.nn import functional as F

from .normalization import residual_layer_norm
from .rms_norm import residual_rms_norm

# How a block exposes a sublayer or norm: an attribute name, or a function of
# the block (and, for sublayers, the normalized input).
Accessor = Union[str, Callable]


def _check_norm(norm: nn.Module, hidden: int) -> None:
    if not isinstance(norm, (nn.LayerNorm, nn.RMSNorm)):
        raise TypeError(
            f"expected torch.nn.LayerNorm or torch.nn.RMSNorm, got {type(norm).__name__}")
    kind = "LayerNorm" if isinstance(norm, nn.LayerNorm) else "RMSNorm"
    if tuple(norm.normalized_shape) != (hidden,):
        raise ValueError(
            f"{kind} normalizes {tuple(norm.normalized_shape)}, the residual stream has "
            f"hidden size {hidden}")
    if norm.weight is None or (kind == "LayerNorm" and norm.bias is None):
        raise ValueError(f"{kind} needs elementwise affine weight"
                         + (" and bias" if kind == "LayerNorm" else ""))


def _rms_eps(norm: nn.RMSNorm, dtype: torch.dtype) -> float:
    """The module's eps. Its default, None, is the epsilon of the type that PyTorch
    computes the norm of a ``dtype`` stream in: fp32's for 16-bit streams as well."""
    if norm.eps is not None:
        return norm.eps
    return torch.finfo(torch.promote_types(dtype, torch.float32)).eps


def _rms_norm(x, branch, norm: nn.RMSNorm, dropout_p, training, implementation, normalized_dtype,
              checkpoint_dtype):
    if branch is not None and training and dropout_p != 0.0:
        branch = F.dropout(branch, dropout_p, True)
    return residual_rms_norm(x, branch, norm.weight, _rms_eps(norm, x.dtype),
                             implementation=implementation, normalized_dtype=normalized_dtype,
                             checkpoint_dtype=checkpoint_dtype)


def _refuse_checkpoint(checkpoint_dtype) -> None:
    if checkpoint_dtype is not None:
        raise ValueError("checkpoint_dtype needs torch.nn.RMSNorm modules")


def residual_norm(x, branch, norm: Union[nn.LayerNorm, nn.RMSNorm], dropout_p: float = 0.0,
                  training: bool = True, *, implementation: str = "auto", normalized_dtype=None,
                  checkpoint_dtype=None):
    """``x + dropout(branch)`` followed by ``norm``, as one fused operation.

    Returns ``(updated, normalized)`` like ``residual_layer_norm``, or like
    ``residual_rms_norm`` for an ``nn.RMSNorm`` (whose dropout, if any, is a
    separate ``F.dropout``); ``norm`` supplies weight, bias and eps and keeps its
    parameters (and their ``state_dict`` keys) in the caller's model.
    ``checkpoint_dtype`` is ``residual_rms_norm``'s.
    """
    _check_norm(norm, x.shape[-1])
    if isinstance(norm, nn.RMSNorm):
        return _rms_norm(x, branch, norm, dropout_p, training, implementation, normalized_dtype,
                         checkpoint_dtype)
    _refuse_checkpoint(checkpoint_dtype)
    return residual_layer_norm(
        x, branch, norm.weight, norm.bias, dropout_p=dropout_p, eps=norm.eps,
        training=training, implementation=implementation, normalized_dtype=normalized_dtype)


def _module(block: nn.Module, accessor: Accessor) -> nn.Module:
    return getattr(block, accessor) if isinstance(accessor, str) else accessor(block)


def _sublayer(block: nn.Module, accessor: Accessor, hidden_states):
    if isinstance(accessor, str):
        return getattr(block, accessor)(hidden_states)
    return accessor(block, hidden_states)


def prenorm_forward(
    x: torch.Tensor,
    blocks: Sequence[nn.Module],
    final_norm: Union[nn.LayerNorm, nn.RMSNorm],
    *,
    dropout_p: float = 0.0,
    training: bool = True,
    attention: Accessor = "attn",
    mlp: Accessor = "mlp",
    ln1: Accessor = "ln_1",
    ln2: Accessor = "ln_2",
    implementation: str = "auto",
    normalized_dtype=None,
    checkpoint_dtype=None,
):
    """Run pre-norm blocks with fused residual LayerNorms; returns ``(x, out)``.

    ``x`` is the fp32 residual stream after the last block and ``out`` the
    final norm of it. ``attention`` and ``mlp`` name each block's sublayers
    (attribute names, called with the normalized input, or functions
    ``f(block, normalized)``); they must return the sublayer output *before*
    its residual dropout, which the fused operation applies with
    ``dropout_p``. ``ln1`` and ``ln2`` name the blocks' LayerNorms (attribute
    names or functions ``f(block)``). ``normalized_dtype`` (fp16 / bf16)
    rounds every normalized output, including ``out``, for half-precision
    sublayers; the residual stream stays fp32.

    The norms may be ``nn.RMSNorm`` modules instead. The residual stream is then
    of ``x``'s own type, fp32, fp16 or bf16, which is also the normalized
    outputs' without ``normalized_dtype``, and ``checkpoint_dtype=torch.int8``
    keeps each norm's input for the backward in 8 bits
    (``residual_rms_norm``), so that no norm keeps the stream itself alive.
    """
    if len(blocks) == 0:
        raise ValueError("prenorm_forward needs at least one block")
    hidden = x.shape[-1]
    first = _module(blocks[0], ln1)
    _check_norm(first, hidden)
    options = dict(implementation=implementation, normalized_dtype=normalized_dtype,
                   checkpoint_dtype=checkpoint_dtype)
    if isinstance(first, nn.RMSNorm):
        x, normalized = _rms_norm(x, None, first, 0.0, training, **options)
    else:
        _refuse_checkpoint(checkpoint_dtype)
        normalized = F.layer_norm(x, (hidden,), first.weight, first.bias, first.eps)
        if normalized_dtype is not None:
            normalized = normalized.to(normalized_dtype)
    for index, block in enumerate(blocks):
        x, normalized = residual_norm(x, _sublayer(block, attention, normalized),
                                      _module(block, ln2), dropout_p, training, **options)
        following = _module(blocks[index + 1], ln1) if index + 1 < len(blocks) else final_norm
        x, normalized = residual_norm(x, _sublayer(block, mlp, normalized), following,
                                      dropout_p, training, **options)
    return x, normalized


__all__ = ["prenorm_forward", "residual_norm"]
