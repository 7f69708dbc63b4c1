"""The root-mean-square norm operators in 64 bits, and how far fp32 kernels may
be from them.

The definition (``include/rln.h``) rounds at three kinds of places, which this
reference rounds too: the new stream to x's type, the 8-bit codes, and each
factor of a code (one fp32 division and one fp32 product). Codes and the
stream are therefore compared bit for bit. Everything else is evaluated in float64
and compared within bounds from fp32 error propagation, u = 2^-24:

* a row's sum of squares: products and at most 16 + 6 + 16 additions (a lane's
  columns, the wave's lanes, the row's waves) of positive terms, 40 u; rstd: half
  of it, the sum's own division, root and quotient, at most 25 u; normalized: two
  products more, 27 u, taken as 32 u relative to the value;
* a gradient g = gu + r (p - unit c): c, a sum of 38 signed additions of
  terms each 30 u off, is off by 70 u * mean|p unit|; with the products and the
  outer additions every term is within 128 u of its magnitude:
  128 u (|gu| + r (|p| + |unit| mean|p unit|));
* the weight's gradient: terms 30 u off, added along at most `depth` additions:
  (32 + depth) u * sum|gy unit|;
* a last rounding to a type: half a step, finfo(t).eps / 2 of the value (and of
  what the value may be off by), or half of the smallest subnormal.
"""

from __future__ import annotations

import torch

U = 2.0 ** -24
TOP = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}
TINY = 2.0 ** -100
SUBNORMAL = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}


def rounding(value, off, dtype):
    """`off` and the rounding of a value that far off to `dtype`."""
    return off + (value.abs() + off) * (torch.finfo(dtype).eps / 2) + SUBNORMAL[dtype] / 2


def update(x, branch):
    return x if branch is None else (x.float() + branch.float()).to(x.dtype)


def rstd_of(u, eps):
    return 1.0 / (u.double().square().mean(-1, keepdim=True) + eps).sqrt()


def normalized(u, weight, eps):
    return u.double() * rstd_of(u, eps) * weight.double()


def normalized_bound(value, dtype):
    return rounding(value, 32 * U * value.abs(), dtype)


def spread(groups, group, hidden):
    return groups.repeat_interleave(group, -1)[..., :hidden]


def codes(values, group, dtype):
    """(codes, maxima) of fp32 values: one fp32 division and one fp32 product."""
    parts = values.split(group, -1)
    largest = torch.stack([part.abs().amax(-1) for part in parts], -1)
    largest = largest.clamp(min=TINY)
    inverse = torch.full_like(largest, TOP[dtype]) / largest
    steps = values * spread(inverse, group, values.shape[-1])
    steps = steps.clamp(-TOP[dtype], TOP[dtype])
    return (steps.round() if dtype == torch.int8 else steps).to(dtype), largest


def quantized(u, weight, eps, group, dtype):
    """(codes, scale in 64 bits); group None is the whole row."""
    values = u.float() * weight.float()
    found, largest = codes(values, group or values.shape[-1], dtype)
    return found, largest.double() / TOP[dtype] * rstd_of(u, eps)


def checkpoint(u):
    """(codes, fp32 scale, what the backward reads for u)."""
    found, largest = codes(u.float(), 128, torch.int8)
    scale = largest / torch.full_like(largest, 127.0)
    return found, scale, found.float() * spread(scale, 128, u.shape[-1])


def gradients(u, kept, weight, eps, grad_updated, grad_normalized):
    """(g, grad_weight) in 64 bits and the magnitudes of their bounds."""
    r = rstd_of(u, eps)
    unit, w = kept.double() * r, weight.double()
    gu = 0.0 if grad_updated is None else grad_updated.double()
    gy = grad_normalized.double()
    p = gy * w
    g = gu + r * (p - unit * (p * unit).mean(-1, keepdim=True))
    size = abs(gu) + r * (p.abs() + unit.abs() * (p * unit).abs().mean(-1, keepdim=True))
    terms = (gy * unit).reshape(-1, u.shape[-1])
    return g, terms.sum(0), size, terms.abs().sum(0)


def gradient_bound(g, size, dtype):
    return rounding(g, 128 * U * size, dtype)


def weight_bound(value, size, depth, dtype):
    return rounding(value, (32 + depth) * U * size, dtype)


def assert_within(actual, expected, bound, what):
    actual = actual.detach().cpu().double()
    assert actual.shape == expected.shape, (what, actual.shape, expected.shape)
    off = (actual - expected).abs()
    bad = ~(off <= bound)
    assert not bad.any(), (
        f"{what}: {int(bad.sum())} of {bad.numel()} values off, the first by "
        f"{off[bad][0].item():.3e} against {bound.expand_as(off)[bad][0].item():.3e}")


def same_bits(a, b):
    """Equal values bit for bit, NaNs included (any type of 1, 2 or 4 bytes)."""
    kind = {1: torch.uint8, 2: torch.int16, 4: torch.int32}[a.element_size()]
    return torch.equal(a.detach().cpu().contiguous().view(kind),
                       b.detach().cpu().contiguous().view(kind))
