"""Graphs recorded by torch.jit.trace and make_fx hold the root-mean-square norm
operators themselves, not the allocations of one call's outputs."""

import warnings

import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx

import rms_reference as reference
from gfx1010_kernels import _C, dequantize, residual_rms_norm, residual_rms_norm_quantized

pytestmark = pytest.mark.gpu
EPS = 1e-6
MODES = ["auto", "gfx950", "torch"]


def make(seed=0, rows=5, hidden=200):
    generator = torch.Generator().manual_seed(seed)
    x, branch = (torch.randn(rows, hidden, generator=generator).cuda() for _ in range(2))
    return x, branch, torch.rand(hidden, generator=generator).cuda()


def functions(implementation, checkpoint=None):
    def norm(x, branch, weight):
        return residual_rms_norm(x, branch, weight, EPS, implementation=implementation,
                                 checkpoint_dtype=checkpoint)

    def first(x, branch, weight):
        return residual_rms_norm(x, None, weight, EPS, implementation=implementation)[1] + branch

    def eight(x, branch, weight):
        _, codes, scale = residual_rms_norm_quantized(x, branch, weight, EPS, dtype=torch.int8,
                                                      group_size=64,
                                                      implementation=implementation)
        return codes, scale, dequantize(codes, scale, group_size=64,
                                        implementation=implementation)
    return norm, first, eight


def check_same(found, expected):
    found, expected = (t if isinstance(t, (tuple, list)) else (t,) for t in (found, expected))
    assert len(found) == len(expected)
    for a, b in zip(found, expected):
        assert a.dtype == b.dtype and reference.same_bits(a, b)


def spoil():
    """Memory that a later allocation of these sizes finds."""
    torch.cuda.empty_cache()
    junk = [torch.full((1 << 18,), float("nan"), device="cuda") for _ in range(4)]
    del junk


@pytest.mark.parametrize("implementation", MODES)
@pytest.mark.parametrize("which", [0, 1, 2])
def test_jit_trace(implementation, which):
    function = functions(implementation)[which]
    residual_rms_norm(*make(), EPS)  # the device is known to be ready
    with torch.no_grad(), warnings.catch_warnings():
        warnings.simplefilter("ignore", torch.jit.TracerWarning)
        traced = torch.jit.trace(function, make())
        for seed, rows in ((1, 5), (2, 5), (3, 9)):
            if rows != 5 and implementation == "torch" and which == 2:
                continue  # a traced decomposition holds its sizes
            inputs = make(seed, rows)
            spoil()
            found, expected = traced(*inputs), function(*inputs)
            if implementation == "torch":  # whose operations PyTorch may fuse: fp32 roundings
                for a, b in zip(found, expected):
                    torch.testing.assert_close(a, b, rtol=64 * reference.U, atol=64 * reference.U)
            else:
                check_same(found, expected)


@pytest.mark.parametrize("implementation", MODES)
@pytest.mark.parametrize("which", [0, 1, 2])
@pytest.mark.parametrize("mode", ["real", "fake", "symbolic"])
def test_make_fx(implementation, which, mode):
    function = functions(implementation)[which]
    residual_rms_norm(*make(), EPS)
    with torch.no_grad():
        graph = make_fx(function, tracing_mode=mode)(*make())
        for seed in (1, 2):
            inputs = make(seed)
            spoil()
            check_same(graph(*inputs), function(*inputs))
        if implementation != "torch":
            assert any("gfx1010_kernels" in str(node.target) for node in graph.graph.nodes)


@pytest.mark.parametrize("checkpoint", [None, torch.int8])
@pytest.mark.parametrize("pre_dispatch", [False, True])
def test_make_fx_of_a_training_step(checkpoint, pre_dispatch):
    norm = functions("auto", checkpoint)[0]

    def step(*leaves):
        outputs = norm(*leaves)
        loss = outputs[0].sin().sum() + outputs[1].square().sum()
        return [*outputs, *torch.autograd.grad(loss, leaves)]

    def leaves(seed):
        return [t.requires_grad_() for t in make(seed)]

    if pre_dispatch:  # records the forward alone: autograd runs below it
        graph = make_fx(norm, pre_dispatch=True)(*make())
        check_same(graph(*make(1)), norm(*make(1)))
        return
    graph = make_fx(step)(*leaves(0))
    for seed in (1, 2):
        found, expected = graph(*leaves(seed)), step(*leaves(seed))
        spoil()
        check_same([t.detach() for t in found], [t.detach() for t in expected])


def test_an_eager_graph_cannot_be_recorded_from_its_middle():
    leaves = [t.requires_grad_() for t in make()]
    loss = residual_rms_norm(*leaves, EPS)[1].square().sum()
    with pytest.raises(RuntimeError, match="recorded into a graph"):
        make_fx(lambda scale: torch.autograd.grad(loss * scale, leaves, retain_graph=True))(
            torch.ones((), device="cuda"))
    grads = torch.autograd.grad(loss, leaves)
    assert all(g.isfinite().all() for g in grads)


def test_the_extension_itself_refuses_to_be_recorded():
    x, branch, weight = make()
    codes = torch.zeros(5, 200, dtype=torch.int8, device="cuda")
    scale = torch.ones(5, 1, device="cuda")
    for call in (lambda t: _C.residual_rms_norm(t, branch, weight, EPS, None, False)[1],
                 lambda t: _C.residual_rms_norm_quantized(t, branch, weight, EPS, torch.int8,
                                                          0)[2],
                 lambda t: _C.dequantize(codes, scale, 0, torch.float32) + t):
        with pytest.raises(RuntimeError, match="recorded into a graph"):
            torch.jit.trace(call, (x,), check_trace=False)
        with pytest.raises(RuntimeError, match="recorded into a graph"):
            make_fx(call)(x)
        call(x)


@pytest.mark.parametrize("checkpoint", [None, torch.int8])
@pytest.mark.parametrize("traced_with_grad", [False, True])
def test_gradients_through_a_traced_call(checkpoint, traced_with_grad):
    norm = functions("auto", checkpoint)[0]
    with torch.set_grad_enabled(traced_with_grad):
        traced = torch.jit.trace(norm, tuple(t.requires_grad_(traced_with_grad) for t in make()))
    for seed, rows in ((1, 5), (2, 5), (3, 2000)):
        results = []
        for call in (traced, norm):
            leaves = [t.requires_grad_() for t in make(seed, rows)]
            outputs = call(*leaves)
            loss = outputs[0].sin().sum() + outputs[1].square().sum()
            results.append([*outputs, *torch.autograd.grad(loss, leaves)])
        check_same(*([t.detach() for t in r] for r in results))
