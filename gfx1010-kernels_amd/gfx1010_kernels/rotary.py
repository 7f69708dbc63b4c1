"""Rotary positions of query and key heads, with the root-mean-square norm of each head.

The reference has no such operator; names, ``implementation`` modes, warnings
and errors here follow ``residual_rms_norm``. :func:`rms_norm_rotary` is what stands
between a joint projection and attention: the heads' own norms (where they have
weights), then the rotation of pairs of values by angles that grow with the token's
position, along one axis (text) or up to four (time, height and width of images and
video), in one pass over queries and keys. :func:`rotary_inverse_frequencies` makes the
angles' table.
"""

from __future__ import annotations

import torch

from ._normalization_native import TARGET_ARCHITECTURE, _extension, graph_recorded
from ._ops import rms_norm_rotary_op
from .normalization import NO_TANGENTS, has_tangent, residual_layer_norm_status
from .rms_norm import (
    STREAM_DTYPES,
    _check_implementation,
    _native_or_reason,
    _READY_DEVICES,
    _rstd,
    _STRICT_NATIVE,
    _warn,
    _wide,
)

MAX_HEAD_SIZE = 256
MAX_HEADS = 1 << 16
MAX_AXES = 4
MAX_TOKENS = (1 << 30) - 1
POSITION_DTYPES = (torch.int64, torch.int32, torch.float32)
FREQUENCY_DTYPES = (torch.float32, torch.float64)
ARRANGEMENTS = ("blocks", "cyclic")
_NO_TABLE_GRADIENTS = "positions and inverse_frequencies have no gradient"
_WHAT = "rotary RMSNorm"


def rotary_inverse_frequencies(sections, base=10000.0, *, shared=True, device=None,
                               dtype=torch.float64):
    """Angles per unit of position, one for each pair of :func:`rms_norm_rotary`.

    ``sections`` are the pairs of each axis, ``(pairs,)`` for a single axis. With
    ``shared`` one ladder runs over all pairs, ``base ** (-i / sum(sections))``; without,
    each axis has a ladder of its own over its section, for sections in blocks.
    """
    sections = tuple(sections)
    if not sections or any(section < 0 for section in sections) or sum(sections) == 0:
        raise ValueError("sections must be numbers of pairs, at least one in all")
    counts = (sum(sections),) if shared else sections
    ladders = [torch.arange(count, dtype=torch.float64) / max(1, count) for count in counts]
    return (float(base) ** -torch.cat(ladders)).to(device=device, dtype=dtype)


def axis_of_pairs(sections, arrangement="blocks"):
    """The axis whose position turns each pair, as a list. In ``"blocks"`` the axes
    follow one another; in ``"cyclic"`` axis ``a > 0`` takes its pairs from ``a`` on,
    every ``len(sections)``-th, as far as there are pairs, and axis 0 has the rest."""
    if arrangement == "blocks":
        return [axis for axis, count in enumerate(sections) for _ in range(count)]
    axes = [0] * sum(sections)
    for axis in range(1, len(sections)):
        for place in range(axis, min(len(axes), axis + sections[axis] * len(sections)),
                           len(sections)):
            axes[place] = axis
    return axes


# The PyTorch decomposition.

def _torch_angles(positions, frequencies, sections, arrangement):
    """[..., 1, pairs], in fp64."""
    if sections is None:
        angles = positions.double().unsqueeze(-1) * frequencies.double()
    else:
        axes = torch.tensor(axis_of_pairs(sections, arrangement), device=positions.device)
        angles = positions.double().index_select(0, axes).movedim(0, -1) * frequencies.double()
    return angles.unsqueeze(-2)


def _torch_turn(heads, weight, cosine, sine, interleaved, eps):
    values = _wide(heads)
    if weight is not None:
        values = values * _rstd(values, eps) * _wide(weight)
    pairs = cosine.shape[-1]
    cosine, sine = cosine.to(values.dtype), sine.to(values.dtype)
    turned, rest = values[..., :2 * pairs], values[..., 2 * pairs:]
    if interleaved:
        first, second = turned[..., 0::2], turned[..., 1::2]
    else:
        first, second = turned[..., :pairs], turned[..., pairs:]
    first, second = first * cosine - second * sine, first * sine + second * cosine
    if interleaved:
        turned = torch.stack([first, second], -1).flatten(-2)
    else:
        turned = torch.cat([first, second], -1)
    return torch.cat([turned, rest], -1).to(heads.dtype)


def _torch_rotary(q, k, positions, frequencies, sections, arrangement, interleaved, q_weight,
                  k_weight, eps):
    angles = _torch_angles(positions, frequencies, sections, arrangement)
    cosine, sine = angles.cos(), angles.sin()
    return (_torch_turn(q, q_weight, cosine, sine, interleaved, eps),
            None if k is None else _torch_turn(k, k_weight, cosine, sine, interleaved, eps))


# Checks and dispatch.

def _broadcasts(sizes, over):
    missing = len(over) - len(sizes)
    return missing >= 0 and all(size in (1, whole) for size, whole in zip(sizes, over[missing:]))


def _whole_sections(sections):
    """``sections`` as a tuple of ints; any sequence of whole numbers."""
    if sections is None:
        return None
    whole = tuple(int(section) for section in sections)
    if not whole:
        raise ValueError("sections must hold at least one number of pairs")
    if any(own != section for own, section in zip(whole, sections)):
        raise ValueError("sections must be whole numbers of pairs")
    return whole


def _check_shapes(q, k, positions, frequencies, sections, arrangement, q_weight, k_weight):
    """What no implementation takes: tensors that do not fit one another."""
    if arrangement not in ARRANGEMENTS:
        raise ValueError("arrangement must be 'blocks' or 'cyclic'")
    if q.ndim < 2 or (k is not None and k.ndim < 2):
        raise ValueError("q and k must have the dimensions [..., heads, size]")
    size = q.shape[-1]
    if k is not None and (k.shape[:-2] != q.shape[:-2] or k.shape[-1] != size
                          or k.dtype != q.dtype):
        raise ValueError("q and k must have the same tokens, head size and type")
    if k is None and k_weight is not None:
        raise ValueError("k_weight needs k")
    if any(weight is not None and weight.shape != (size,) for weight in (q_weight, k_weight)):
        raise ValueError("q_weight and k_weight must match the head size")
    if frequencies.ndim != 1 or not 2 <= 2 * frequencies.shape[0] <= size:
        raise ValueError("inverse_frequencies must hold 1 to size / 2 values")
    tokens = tuple(positions.shape)
    if sections is not None:
        if any(section < 0 for section in sections) or sum(sections) != frequencies.shape[0]:
            raise ValueError("sections must add up to the number of inverse_frequencies")
        if positions.ndim < 1 or tokens[0] != len(sections):
            raise ValueError("positions must have one row for each section")
        tokens = tokens[1:]
    if not _broadcasts(tokens, tuple(q.shape[:-2])):
        raise ValueError("positions must broadcast over the tokens")


def _tables_have_gradients(positions, frequencies):
    return torch.is_grad_enabled() and (positions.requires_grad or frequencies.requires_grad)


def _input_reason(q, k, positions, frequencies, sections, q_weight, k_weight, eps):
    """Why the native kernels cannot serve inputs that fit one another, or None."""
    heads = [tensor for tensor in (q, k) if tensor is not None]
    weights = [tensor for tensor in (q_weight, k_weight) if tensor is not None]
    tensors = [*heads, positions, frequencies, *weights]
    if not all(tensor.is_cuda for tensor in tensors):
        return "all tensors must be HIP tensors"
    if any(tensor.device != q.device for tensor in tensors):
        return "all tensors must be on the same HIP device"
    if has_tangent(*tensors):
        return NO_TANGENTS
    if not 1 <= q.shape[-1] <= MAX_HEAD_SIZE:
        return f"heads must have 1 to {MAX_HEAD_SIZE} values"
    if any(tensor.dtype not in STREAM_DTYPES for tensor in (*heads, *weights)):
        return "q, k and their weights must use float16, bfloat16 or float32"
    if any(tensor.shape[-2] > MAX_HEADS for tensor in heads):
        return f"at most {MAX_HEADS} heads are supported"
    if frequencies.dtype not in FREQUENCY_DTYPES:
        return "inverse_frequencies must use float32 or float64"
    if positions.dtype not in POSITION_DTYPES:
        return "positions must use int64, int32 or float32"
    if sections is not None and len(sections) > MAX_AXES:
        return f"at most {MAX_AXES} axes are supported"
    if _tables_have_gradients(positions, frequencies):
        return _NO_TABLE_GRADIENTS
    if q.shape[:-2].numel() > MAX_TOKENS:
        return "too many tokens"
    if not eps >= 0.0:
        return "eps must not be negative"
    return None


def rms_norm_rotary(
    q,
    k,
    positions,
    inverse_frequencies,
    *,
    sections=None,
    arrangement="blocks",
    interleaved=False,
    q_weight=None,
    k_weight=None,
    eps=1e-6,
    implementation="auto",
):
    """Norms the heads of ``q`` and ``k`` and turns them by their tokens' positions;
    returns ``(q, k)``, new dense tensors of the same shapes and type.

    ``q`` and ``k`` are ``[..., heads, size]`` with the same tokens and as many heads as
    each has (``k`` may be None, and is then returned as None); views, such as parts of a
    joint projection, are read in place. With ``q_weight`` or ``k_weight`` (``[size]``) each
    head is divided by its root mean square and multiplied by the weight first.

    ``inverse_frequencies`` (``[pairs]``, fp32 or fp64) turn the first ``2 * pairs`` values
    of a head, pair ``i`` being values ``i`` and ``i + pairs`` or, with ``interleaved``, ``2i``
    and ``2i + 1``; the rest stays. The angle is ``positions * inverse_frequencies[i]``, taken
    in fp64, so that far positions keep their angles. ``positions`` (int64, int32 or fp32)
    broadcast over the tokens; with ``sections`` they are ``[axes, ...]``, and ``sections``
    gives the pairs of each axis, up to four, in ``arrangement`` ``"blocks"`` or ``"cyclic"``
    (:func:`axis_of_pairs`).

    Supports first-order autograd for the heads and their weights (summed in fp32 in a
    fixed order: bitwise reproducible), HIP graph capture, ``torch.compile``,
    ``torch.jit.trace`` and ``make_fx``; inputs with a forward-mode tangent, and positions or
    frequencies that require a gradient, take the PyTorch path (the native modes raise, in
    every kind of graph too). The kernels serve heads of up to 256 values in fp32, fp16 and
    bf16. The graph keeps the heads only where they are normed, and nothing else of their
    size.
    """
    ready = q.is_cuda and q.get_device() in _READY_DEVICES
    if (implementation == "auto" and ready and arrangement in ARRANGEMENTS
            and (sections is None or len(sections) > 0) and not torch.compiler.is_compiling()):
        try:
            result = _extension()[0].rms_norm_rotary_if_supported(
                q, k, positions, inverse_frequencies, () if sections is None else sections,
                arrangement == "cyclic", interleaved, q_weight, k_weight, float(eps))
        except TypeError:  # sections of another kind than the extension takes, among others
            if sections is None:
                raise
            result = None
        if result is not None:
            return result
    _check_implementation(implementation, _WHAT)
    sections = _whole_sections(sections)
    args = (q, k, positions, inverse_frequencies)
    _check_shapes(*args, sections, arrangement, q_weight, k_weight)
    eps = float(eps)
    plain = (*args, sections, arrangement, bool(interleaved), q_weight, k_weight, eps)
    given = (*args, list(sections or ()), arrangement == "cyclic", bool(interleaved), q_weight,
             k_weight, eps)

    def reason_of():
        return _input_reason(*args, sections, q_weight, k_weight, eps)

    strict = implementation in _STRICT_NATIVE
    if implementation == "torch":
        return _torch_rotary(*plain)
    if torch.compiler.is_compiling():
        reason = reason_of()
        if strict and reason in (NO_TANGENTS, _NO_TABLE_GRADIENTS):
            raise RuntimeError(f"{TARGET_ARCHITECTURE} native {_WHAT} is unavailable: {reason}")
        return rms_norm_rotary_op(*given) if strict or reason is None else _torch_rotary(*plain)
    if q.is_cuda and graph_recorded():
        if strict and _tables_have_gradients(positions, inverse_frequencies):
            raise RuntimeError(
                f"{TARGET_ARCHITECTURE} native {_WHAT} is unavailable: {_NO_TABLE_GRADIENTS}")
        if not strict:
            reason = (_extension()[0].rotary_inputs_refusal(*given) if torch.jit.is_tracing()
                      else reason_of())
        return rms_norm_rotary_op(*given) if strict or reason is None else _torch_rotary(*plain)
    native, reason = _native_or_reason(q, reason_of, implementation, _WHAT)
    if native is None:
        _warn(reason, _WHAT)
        return _torch_rotary(*plain)
    return native.rms_norm_rotary(*given)


def can_use_rms_norm_rotary(q, k, positions, inverse_frequencies, *, sections=None,
                            arrangement="blocks", interleaved=False, q_weight=None, k_weight=None,
                            eps=1e-6):
    """True when ``implementation="auto"`` runs natively."""
    try:
        sections = _whole_sections(sections)
        _check_shapes(q, k, positions, inverse_frequencies, sections, arrangement, q_weight,
                      k_weight)
    except ValueError:
        return False
    reason = _input_reason(q, k, positions, inverse_frequencies, sections, q_weight, k_weight,
                           float(eps))
    return reason is None and residual_layer_norm_status(q.device).available


__all__ = [
    "axis_of_pairs",
    "can_use_rms_norm_rotary",
    "rms_norm_rotary",
    "rotary_inverse_frequencies",
]
