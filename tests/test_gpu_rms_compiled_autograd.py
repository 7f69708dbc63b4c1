"""Compiled autograd over the root-mean-square norm's node: the gradients of the
eager engine, bit for bit."""

import itertools

import pytest
import torch
import torch._dynamo.compiled_autograd as compiled_autograd

import rms_reference as reference
from gfx1010_kernels import residual_rms_norm

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def leaves(seed, x_dtype, branch_dtype, added=True, needs=(True, True, True), hidden=200):
    generator = torch.Generator().manual_seed(seed)
    x, branch = (torch.randn(6, hidden, generator=generator) for _ in range(2))
    weight = 1.0 + 0.1 * torch.randn(hidden, generator=generator)
    made = [x.to("cuda", x_dtype), branch.to("cuda", branch_dtype) if added else None,
            weight.cuda()]
    return [t if t is None else t.requires_grad_(need) for t, need in zip(made, needs)]


def grads_of(inputs, function, backend):
    torch._dynamo.reset()
    if backend is None:
        function(*inputs).backward()
    else:
        with compiled_autograd._enable(torch.compile(backend=backend)):
            function(*inputs).backward()
    return [None if t is None else t.grad for t in inputs]


def check(function, backend="eager", **options):
    for seed in (0, 1):  # the second one from the compiled graph's cache
        expected = grads_of(leaves(seed, **options), function, None)
        found = grads_of(leaves(seed, **options), function, backend)
        for a, b in zip(found, expected):
            assert (a is None) == (b is None)
            assert a is None or (a.dtype == b.dtype and reference.same_bits(a, b))


@pytest.mark.parametrize("backend", ["eager", "aot_eager"])
@pytest.mark.parametrize("checkpoint", [None, torch.int8])
@pytest.mark.parametrize("added", [True, False])
@pytest.mark.parametrize("x_dtype,branch_dtype", [(F32, F32), (F32, BF16), (BF16, BF16), (F16, F32)])
def test_types(x_dtype, branch_dtype, added, checkpoint, backend):
    def function(x, branch, weight):
        updated, normalized = residual_rms_norm(x, branch, weight, checkpoint_dtype=checkpoint)
        return updated.float().sin().sum() + normalized.float().square().sum()

    check(function, backend, x_dtype=x_dtype, branch_dtype=branch_dtype, added=added)


@pytest.mark.parametrize("checkpoint", [None, torch.int8])
@pytest.mark.parametrize("outputs", [(0,), (1,)])
@pytest.mark.parametrize("needs", [n for n in itertools.product([True, False], repeat=3) if any(n)])
def test_parts(needs, outputs, checkpoint):
    def function(*inputs):
        results = residual_rms_norm(*inputs, checkpoint_dtype=checkpoint)
        return sum(results[i].float().square().sum() for i in outputs)

    if outputs == (0,) and not (needs[0] or needs[1]):
        pytest.skip("the sum alone has no gradient to the weight")
    check(function, x_dtype=F32, branch_dtype=BF16, needs=needs)


@pytest.mark.parametrize("checkpoint", [None, torch.int8])
def test_a_stack_whose_leaves_come_again(checkpoint):
    def function(x, branch, weight):
        total = 0.0
        for _ in range(3):
            x, normalized = residual_rms_norm(x, branch, weight, checkpoint_dtype=checkpoint)
            branch = normalized.sin() + branch
            total = total + normalized.square().sum()
        return total + residual_rms_norm(x, None, weight, checkpoint_dtype=checkpoint)[1].sum()

    check(function, x_dtype=F32, branch_dtype=F32)


def test_a_compiled_step():
    """Forward and backward compiled together."""
    def function(x, branch, weight):
        updated, normalized = residual_rms_norm(x, branch, weight)
        return updated.sin().sum() + normalized.square().sum()

    expected = grads_of(leaves(3, F32, BF16), function, None)
    inputs = leaves(3, F32, BF16)
    torch._dynamo.reset()
    with compiled_autograd._enable(torch.compile(backend="aot_eager")):
        torch.compile(function, backend="aot_eager")(*inputs).backward()
    for a, b in zip(inputs, expected):
        assert reference.same_bits(a.grad, b)


@pytest.mark.parametrize("checkpoint", [None, torch.int8])
def test_other_row_counts_after_the_first(checkpoint):
    """One compiler over calls of several sizes, whose graphs it may make dynamic."""
    def function(x, branch, weight):
        updated, normalized = residual_rms_norm(x, branch, weight, checkpoint_dtype=checkpoint)
        return updated.float().sin().sum() + normalized.float().square().sum()

    def inputs(rows, hidden):
        generator = torch.Generator("cuda").manual_seed(rows)
        return [torch.randn(shape, device="cuda", generator=generator).requires_grad_()
                for shape in ((rows, hidden), (rows, hidden), (hidden,))]

    torch._dynamo.reset()
    compiler = torch.compile(backend="eager")
    for rows, hidden in ((6, 200), (7, 200), (9, 200), (9, 96), (2000, 200)):
        expected, found = inputs(rows, hidden), inputs(rows, hidden)
        function(*expected).backward()
        with compiled_autograd._enable(compiler):
            function(*found).backward()
        assert all(reference.same_bits(a.grad, b.grad) for a, b in zip(found, expected))
