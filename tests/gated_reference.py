"""The gated residual norm in 64 bits, and how far fp32 kernels may be from it.

Like rms_reference.py (whose bounds of a norm are used), with u = 2^-24. The
reference takes the kernels' own rounded stream for what depends on it.

* branch_rstd is within 25 u, b = branch * branch_rstd within 26 u; c =
  branch_scale * gate * branch_weight is three roundings off (the constant's own
  among them); so c * b is within 30 u, residual_scale * x within 2 u, and their
  sum within 3 u |residual_scale x| + 32 u |c b|, rounded to x's type;
* g, the stream's gradient, is within 128 u of size = |gu| + r (|p| + |v| mean|p v|)
  (rms_reference.py), grad_x within 130 u of |residual_scale| size;
* sum(c g b) is taken as sum(c b (gu + r p)) - r sum(p v) / H * sum(c b v): sums of 38
  additions whose terms are products of factors at most 64 u off altogether, the
  middle one 128 u: within 256 u of M = mean(|c b| (|gu| + r |p|)) + r mean|p v| mean|c b v|;
  grad_branch = rb (c g - b mean(c g b)): within 320 u of rb (|c| size + |b| M);
* the terms of grad_gate and grad_branch_weight are 128 + 26 + 5 u off, those of
  grad_weight 30 u; `depth` additions add depth u of the terms' magnitudes.
"""

from __future__ import annotations

import torch

import rms_reference
from rms_reference import U, rounding


def wide(tensor):
    if tensor is None:
        return torch.ones((), dtype=torch.float64)
    return tensor.detach().cpu().double()


class Call:
    """One call's inputs in 64 bits; `parts` are x, branch, weight, branch_weight, gate."""

    def __init__(self, parts, eps, branch_eps, residual_scale, branch_scale):
        self.parts = parts
        self.x, self.branch, self.weight, self.post, self.gate = (wide(t) for t in parts)
        self.eps, self.rs, self.bs = eps, residual_scale, branch_scale
        self.rb = torch.ones(())
        if parts[3] is not None:
            self.rb = rms_reference.rstd_of(self.branch, branch_eps)
        self.b = self.branch * self.rb
        self.c = self.bs * self.gate * self.post

    def updated(self):
        """(value, how far off an unrounded one may be)"""
        kept, added = self.rs * self.x, self.c * self.b
        return kept + added, U * (3 * kept.abs() + 32 * added.abs())

    def check_forward(self, updated, normalized, dtype, what):
        value, off = self.updated()
        x_type = self.parts[0].dtype
        assert updated.dtype == x_type and normalized.dtype == dtype, what
        rms_reference.assert_within(updated, value, rounding(value, off, x_type),
                                    f"{what}: updated")
        y = wide(updated) * rms_reference.rstd_of(wide(updated), self.eps) * self.weight
        rms_reference.assert_within(normalized, y, rms_reference.normalized_bound(y, dtype),
                                    f"{what}: normalized")

    def gradients(self, updated, grad_updated, grad_normalized):
        """Per input (value, off) in the order of the parts; depth is the rows'
        number and what a block and a reduction add to it."""
        u = wide(updated)
        r = rms_reference.rstd_of(u, self.eps)
        v = u * r
        gu = torch.zeros_like(u) if grad_updated is None else wide(grad_updated)
        gy = torch.zeros_like(u) if grad_normalized is None else wide(grad_normalized)
        p = gy * self.weight
        mean = (p * v).mean(-1, keepdim=True)
        g = gu + r * (p - v * mean)
        size = gu.abs() + r * (p.abs() + v.abs() * (p * v).abs().mean(-1, keepdim=True))
        depth = u.numel() // u.shape[-1] + 100
        result = [(self.rs * g, 130 * U * abs(self.rs) * size)]
        q = self.c * g
        if self.parts[3] is None:
            result.append((q, 140 * U * self.c.abs() * size))
        else:
            value = self.rb * (q - self.b * (q * self.b).mean(-1, keepdim=True))
            cb = self.c * self.b
            m = ((cb.abs() * (gu.abs() + r * p.abs())).mean(-1, keepdim=True)
                 + r * (p * v).abs().mean(-1, keepdim=True) * (cb * v).abs().mean(-1, keepdim=True))
            result.append((value, 320 * U * self.rb * (self.c.abs() * size + self.b.abs() * m)))

        def summed(terms, sizes, index, each):
            like = self.parts[index]
            if like is None:
                return None
            count = u.numel() // max(1, like.numel())
            steps = each + (depth if count > 1 else 0)
            return (terms.expand(u.shape).sum_to_size(like.shape),
                    steps * U * sizes.expand(u.shape).sum_to_size(like.shape))

        result.append(summed(gy * v, (gy * v).abs(), 2, 32))
        each, sizes = self.bs * g * self.b, abs(self.bs) * size * self.b.abs()
        result.append(summed(each * self.gate, sizes * self.gate.abs(), 3, 192))
        result.append(summed(each * self.post, sizes * self.post.abs(), 4, 192))
        return result

    def check_gradients(self, grads, updated, grad_updated, grad_normalized, what):
        """`grads` in the order of the parts; None where not asked for."""
        expected = self.gradients(updated, grad_updated, grad_normalized)
        names = ("x", "branch", "weight", "branch_weight", "gate")
        for name, grad, part, entry in zip(names, grads, self.parts, expected):
            if grad is None:
                continue
            value, off = entry
            assert grad.dtype == part.dtype and grad.shape == part.shape, (what, name)
            rms_reference.assert_within(grad, value, rounding(value, off, part.dtype),
                                        f"{what}: grad of {name}")


def make(shape, dtypes, *, post=True, gate="sample", weight="shared", seed=0):
    """CPU parts (x, branch, weight, branch_weight, gate) from the seed. `gate` and
    `weight` are "none", "shared", "sample", "token" or a shape; `dtypes` the types of
    x, branch, weight, branch_weight and gate."""
    generator = torch.Generator().manual_seed(seed)
    hidden = shape[-1]

    def normal(size, dtype, scale=1.0, mean=0.0):
        return (torch.randn(size, generator=generator) * scale + mean).to(dtype)

    def factor_shape(kind):
        kinds = {"shared": (hidden,), "sample": (*shape[:1], *[1] * (len(shape) - 2), hidden),
                 "token": tuple(shape)}
        return kinds.get(kind, kind)

    x = normal(shape, torch.float32)
    x = (x * (1.0 + 15.0 * (torch.rand(hidden, generator=generator) < 0.02))).to(dtypes[0])
    return (x, normal(shape, dtypes[1], 0.5),
            normal(factor_shape(weight), dtypes[2], 0.1, 1.0),
            normal((hidden,), dtypes[3], 0.1, 1.0) if post else None,
            None if gate == "none" else normal(factor_shape(gate), dtypes[4], 0.5))
