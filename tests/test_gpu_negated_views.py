"""Lazily negated tensors, such as the imaginary part of a conjugate: their memory holds the
values with the other sign."""

import pytest
import torch

from gfx1010_kernels import (
    dequantize,
    gated_residual_rms_norm,
    residual_rms_norm,
    residual_rms_norm_quantized,
    rms_norm_rotary,
)
from rms_reference import same_bits

pytestmark = pytest.mark.gpu


def views(tensor):
    """``tensor`` as such views: dense, and as complex numbers have their parts."""
    yield torch._neg_view(-tensor)
    yield torch.complex(torch.zeros_like(tensor), -tensor).conj().imag


def normal(*shape, seed=0):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed + len(shape))).cuda()


def check(function, tensors, upstream):
    """Each tensor in turn as a view, then the upstream gradients."""
    def step(given, above):
        leaves = [t.detach().requires_grad_() for t in given]
        outputs = function(*leaves)
        return [*outputs, *torch.autograd.grad(outputs, leaves, above)]

    expected = step(tensors, upstream)
    for place in range(len(tensors) + len(upstream)):
        whole = [*tensors, *upstream]
        for view in views(whole[place]):
            assert view.is_neg() and torch.equal(view, whole[place])
            given = [*whole[:place], view, *whole[place + 1:]]
            found = step(given[:len(tensors)], given[len(tensors):])
            assert all(same_bits(a, b) for a, b in zip(found, expected)), place


@pytest.mark.parametrize("hidden", [1, 64])
def test_gated_residual_norm(hidden):
    tensors = [normal(3, hidden, seed=i) for i in range(2)] + [normal(hidden, seed=i)
                                                               for i in (2, 3, 4)]
    check(lambda x, branch, weight, post, gate: gated_residual_rms_norm(
        x, branch, weight, branch_weight=post, gate=gate, implementation="gfx950"),
        tensors, [normal(3, hidden, seed=i) for i in (5, 6)])


@pytest.mark.parametrize("hidden", [1, 64])
def test_residual_rms_norm(hidden):
    x, branch, weight = normal(3, hidden), normal(3, hidden, seed=1), normal(hidden, seed=2)
    check(lambda *given: residual_rms_norm(*given, implementation="gfx950"), [x, branch, weight],
          [normal(3, hidden, seed=i) for i in (3, 4)])
    expected = residual_rms_norm_quantized(x, branch, weight, implementation="gfx950")
    for place, tensor in enumerate((x, branch, weight)):
        for view in views(tensor):
            given = [x, branch, weight]
            given[place] = view
            found = residual_rms_norm_quantized(*given, implementation="gfx950")
            for a, b in zip(found, expected):
                assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    values = dequantize(*expected[1:], dtype=torch.float32)
    for view in views(expected[2]):
        assert same_bits(dequantize(expected[1], view, dtype=torch.float32), values)


def test_rotary_norm_of_heads():
    q, k, qw, kw = normal(5, 4, 16), normal(5, 2, 16), normal(16), normal(16, seed=1)
    positions, frequencies = normal(5, seed=3) * 100, normal(8, seed=4)
    check(lambda q, k, qw, kw: rms_norm_rotary(
        q, k, positions, frequencies, q_weight=qw, k_weight=kw, implementation="gfx950"),
        [q, k, qw, kw], [normal(5, 4, 16, seed=5), normal(5, 2, 16, seed=6)])
    for axes in (None, (5, 3)):
        where = positions if axes is None else torch.stack([positions, positions + 1])
        expected = rms_norm_rotary(q, k, where, frequencies, sections=axes)
        for tables in ([(view, frequencies) for view in views(where)]
                       + [(where, view) for view in views(frequencies)]):
            found = rms_norm_rotary(q, k, *tables, sections=axes, implementation="gfx950")
            assert all(same_bits(a, b) for a, b in zip(found, expected))
