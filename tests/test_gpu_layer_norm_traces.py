"""Graphs recorded by torch.jit.trace and make_fx hold the residual LayerNorm
itself, not the allocations of one call's outputs."""

import warnings

import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx

from gfx1010_kernels import _C, residual_layer_norm

pytestmark = pytest.mark.gpu


def make(seed=0, rows=5, hidden=1024):
    generator = torch.Generator().manual_seed(seed)
    x, branch = (torch.randn(rows, hidden, generator=generator).cuda() for _ in range(2))
    weight, bias = (torch.rand(hidden, generator=generator).cuda() for _ in range(2))
    return x, branch, weight, bias


def spoil():
    """Memory that a later allocation of these sizes finds."""
    torch.cuda.empty_cache()
    junk = [torch.full((1 << 18,), float("nan"), device="cuda") for _ in range(4)]
    del junk


def norm(implementation, dropout_p=0.0):
    def function(*inputs):
        return residual_layer_norm(*inputs, dropout_p, implementation=implementation,
                                   normalized_dtype=torch.bfloat16)
    return function


@pytest.mark.parametrize("dropout_p", [0.0, 0.25])
@pytest.mark.parametrize("implementation", ["auto", "gfx950"])
@pytest.mark.parametrize("hidden", [128, 1024])
def test_jit_trace(implementation, hidden, dropout_p):
    function = norm(implementation, dropout_p)
    residual_layer_norm(*make(), 0.0)  # the device is known to be ready
    with torch.no_grad(), warnings.catch_warnings():
        warnings.simplefilter("ignore", torch.jit.TracerWarning)
        traced = torch.jit.trace(function, make(hidden=hidden), check_trace=dropout_p == 0.0)
        for seed, rows in ((1, 5), (2, 9)):
            inputs = make(seed, rows, hidden)
            results = []
            for call in (traced, function):  # the same masks from the same generator state
                spoil()
                torch.manual_seed(seed)
                results.append(call(*inputs))
            assert all(torch.equal(a, b) for a, b in zip(*results))


@pytest.mark.parametrize("implementation", ["auto", "gfx950"])
@pytest.mark.parametrize("mode", ["real", "fake", "symbolic"])
def test_make_fx(implementation, mode):
    function = norm(implementation)
    residual_layer_norm(*make(), 0.0)
    with torch.no_grad():
        graph = make_fx(function, tracing_mode=mode)(*make())
        spoil()
        assert all(torch.equal(a, b) for a, b in zip(graph(*make(1)), function(*make(1))))
    assert any("rln_forward" in str(node.target) for node in graph.graph.nodes)


def test_make_fx_of_a_training_step():
    def step(*leaves):
        outputs = norm("auto")(*leaves)
        loss = outputs[0].sin().sum() + outputs[1].float().square().sum()
        return [*outputs, *torch.autograd.grad(loss, leaves)]

    def leaves(seed):
        return [t.requires_grad_() for t in make(seed)]

    with torch.random.fork_rng(devices=[0]):
        torch.use_deterministic_algorithms(True)
        try:
            graph = make_fx(step)(*leaves(0))
            found, expected = graph(*leaves(1)), step(*leaves(1))
        finally:
            torch.use_deterministic_algorithms(False)
    assert all(torch.equal(a, b) for a, b in zip(found, expected))


def test_other_sizes_take_the_decomposition():
    """136 columns are no native size: recorded without a warning, as compiled."""
    function = norm("auto")
    inputs = make(hidden=136)
    with torch.no_grad(), warnings.catch_warnings():
        warnings.simplefilter("error", RuntimeWarning)
        warnings.simplefilter("ignore", torch.jit.TracerWarning)
        for graph in (torch.jit.trace(function, inputs, check_trace=False),
                      make_fx(function)(*inputs)):
            for a, b in zip(graph(*inputs), norm("torch")(*inputs)):
                torch.testing.assert_close(a, b)


def test_the_extension_itself_refuses_to_be_recorded():
    x, branch, weight, bias = make()

    def call(t):
        return _C.residual_layer_norm(t, branch, weight, bias, 0.0, 1e-5, True, 192, 64, 64, 1)[1]

    with pytest.raises(RuntimeError, match="recorded into a graph"):
        torch.jit.trace(call, (x,), check_trace=False)
    with pytest.raises(RuntimeError, match="recorded into a graph"):
        make_fx(call)(x)
    leaves = [t.requires_grad_() for t in (x, branch, weight, bias)]
    loss = norm("auto")(*leaves)[1].float().sum()
    with pytest.raises(RuntimeError, match="recorded into a graph"):
        make_fx(lambda scale: torch.autograd.grad(loss * scale, leaves, retain_graph=True))(
            torch.ones((), device="cuda"))
    assert all(g.isfinite().all() for g in torch.autograd.grad(loss, leaves))
