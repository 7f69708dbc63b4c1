"""The rotary norm of heads in 64 bits, and how far fp32 kernels may be from it.

u = 2^-24. rstd of a head: 16 products and at most 12 additions of positive terms, half
of it, the root and the quotient: within 18 u; a normed value within 20 u. Cosine and
sine: the angle's rest is rounded once (at most an eighth of a turn), the
polynomials add about a unit in the last place, and fp64 angles below 2^27 are
2^-25 off: within 3 u in all. A turned value x c - y s is therefore within 28 u of
|x| + |y| (8 u without a norm), and rounded once.

Backward, S = |g1| + |g2| of a pair: t, the gradient turned back, within 8 u S; with n
the normed head, p = t w and c = mean(p n), a sum of 28 signed additions of terms 30 u
off: r (p - n c) within 96 u r (|w| S + |n| mean(|w| S |n|)); the weight's gradient, terms
30 u off added along at most `depth` additions.
"""

from __future__ import annotations

import torch

import rms_reference
from rms_reference import U, rounding


def axes_of(sections, arrangement):
    if sections is None:
        return None
    axes = [axis for axis, count in enumerate(sections) for _ in range(count)]
    if arrangement == "cyclic":
        axes = [0] * len(axes)
        for axis in range(1, len(sections)):
            for turn in range(sections[axis]):
                if axis + turn * len(sections) < len(axes):
                    axes[axis + turn * len(sections)] = axis
    return axes


def angles_of(positions, frequencies, sections, arrangement, tokens):
    """[*tokens, 1, pairs]"""
    positions, frequencies = positions.cpu().double(), frequencies.cpu().double()
    axes = axes_of(sections, arrangement)
    if axes is None:
        picked = positions.expand(tokens).unsqueeze(-1)
    else:
        shape = (len(sections), *[1] * (len(tokens) + 1 - positions.ndim), *positions.shape[1:])
        whole = positions.reshape(shape).expand(len(sections), *tokens)
        picked = torch.stack([whole[axis] for axis in axes], -1)
    return (picked * frequencies).unsqueeze(-2)


def halves(values, pairs, interleaved):
    if interleaved:
        return values[..., 0:2 * pairs:2], values[..., 1:2 * pairs:2]
    return values[..., :pairs], values[..., pairs:2 * pairs]


def joined(first, second, rest, interleaved):
    turned = (torch.stack([first, second], -1).flatten(-2) if interleaved
              else torch.cat([first, second], -1))
    return torch.cat([turned, rest], -1)


def turn(values, angles, interleaved):
    pairs = angles.shape[-1]
    first, second = halves(values, pairs, interleaved)
    c, s = angles.cos(), angles.sin()
    return joined(first * c - second * s, first * s + second * c, values[..., 2 * pairs:],
                  interleaved)


def pair_size(values, pairs, interleaved):
    """|n1| + |n2| at both values of a pair, |n| at the rest."""
    values = values.abs()
    first, second = halves(values, pairs, interleaved)
    both = first + second
    return joined(both, both, values[..., 2 * pairs:], interleaved)


def rstd_of(heads, eps):
    return rms_reference.rstd_of(heads, eps)


def check_forward(output, heads, weight, angles, interleaved, eps, what):
    h = heads.detach().cpu().double()
    scale = 8
    if weight is not None:
        h, scale = h * rstd_of(h, eps) * weight.detach().cpu().double(), 28
    value = turn(h, angles, interleaved)
    off = scale * U * pair_size(h, angles.shape[-1], interleaved)
    assert output.dtype == heads.dtype, what
    rms_reference.assert_within(output, value, rounding(value, off, heads.dtype), what)


def gradients(heads, weight, upstream, angles, interleaved, eps):
    """((grad, off), (grad_weight, off) or None)"""
    g = upstream.detach().cpu().double()
    t = turn(g, -angles, interleaved)
    size = pair_size(g, angles.shape[-1], interleaved)
    if weight is None:
        return (t, 8 * U * size), None
    h, w = heads.detach().cpu().double(), weight.detach().cpu().double()
    r = rstd_of(h, eps)
    n = h * r
    grad = r * (t * w - n * (t * w * n).mean(-1, keepdim=True))
    off = 96 * U * r * (w.abs() * size
                        + n.abs() * (w.abs() * size * n.abs()).mean(-1, keepdim=True))
    count = h.numel() // h.shape[-1]
    terms, sizes = (t * n).flatten(0, -2), (size * n.abs()).flatten(0, -2)
    return (grad, off), (terms.sum(0), (32 + count + 100) * U * sizes.sum(0))


def check_gradients(grad, grad_weight, heads, weight, upstream, angles, interleaved, eps, what):
    one, two = gradients(heads, weight, upstream, angles, interleaved, eps)
    if grad is not None:
        assert grad.dtype == heads.dtype and grad.shape == heads.shape, what
        rms_reference.assert_within(grad, one[0], rounding(*one, heads.dtype), f"{what}: heads")
    if grad_weight is not None:
        assert grad_weight.dtype == weight.dtype, what
        rms_reference.assert_within(grad_weight, two[0], rounding(*two, weight.dtype),
                                    f"{what}: weight")


def make(tokens, q_heads, k_heads, size, dtype, *, pairs=None, axes=1, norm=True, weight_dtype=None,
         seed=0, far=0, position_dtype=torch.int64):
    """CPU tensors (q, k, positions [axes, *tokens], frequencies, q_weight, k_weight)."""
    generator = torch.Generator().manual_seed(seed)
    pairs = size // 2 if pairs is None else pairs

    def normal(shape, kind, scale=1.0, mean=0.0):
        return (torch.randn(shape, generator=generator) * scale + mean).to(kind)

    positions = far + torch.randint(0, 5000, (axes, *tokens), generator=generator)
    positions = positions.to(position_dtype)
    frequencies = (10000.0 ** -(torch.arange(pairs).double() / pairs)).float()
    kind = weight_dtype or dtype
    return (normal((*tokens, q_heads, size), dtype),
            normal((*tokens, k_heads, size), dtype) if k_heads else None, positions, frequencies,
            normal((size,), kind, 0.1, 1.0) if norm else None,
            normal((size,), kind, 0.1, 1.0) if norm and k_heads else None)
