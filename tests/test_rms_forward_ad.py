"""Forward-mode derivatives of the root-mean-square norm operators: carried by the
PyTorch path, which ``"auto"`` takes for inputs with a tangent, and refused by the
kernels, which would drop them."""

import itertools

import pytest
import torch
from torch.autograd import forward_ad

import rms_reference as reference
from gfx1010_kernels import (
    can_use_residual_rms_norm,
    dequantize,
    residual_rms_norm,
    residual_rms_norm_quantized,
)

EPS = 1e-6
HIDDEN = 96
PARTS = ["x", "branch", "weight"]


def make(device, seed=0):
    generator = torch.Generator().manual_seed(seed)
    x, branch, dx, db = (torch.randn(5, HIDDEN, generator=generator) for _ in range(4))
    weight, dw = (torch.randn(HIDDEN, generator=generator) for _ in range(2))
    values = dict(x=x, branch=branch, weight=weight)
    directions = dict(x=dx, branch=db, weight=dw)
    return ({k: v.to(device) for k, v in values.items()},
            {k: v.to(device) for k, v in directions.items()})


def dual(values, directions, moved, requires_grad=False):
    return [forward_ad.make_dual(values[k].clone().requires_grad_(requires_grad), directions[k])
            if k in moved else values[k] for k in PARTS]


def check_tangents(outputs, values, directions, moved):
    """Against the derivative in 64 bits. A tangent is a sum of terms that each take
    a few fp32 operations and, in the mean, HIDDEN signed additions: within
    (HIDDEN + 128) u of the terms' magnitudes, as the gradients' bound."""
    values = {k: v.cpu().double() for k, v in values.items()}
    zero = {k: torch.zeros_like(v) for k, v in values.items()}
    d = {k: directions[k].cpu().double() if k in moved else zero[k] for k in PARTS}
    u, du = values["x"] + values["branch"], d["x"] + d["branch"]
    w, dw = values["weight"], d["weight"]
    r = reference.rstd_of(u, EPS)
    inner = u * r * (u * r * du).mean(-1, keepdim=True)
    size = r * (w.abs() * (du.abs() + u.abs() * r * (u * r * du).abs().mean(-1, keepdim=True))
                + u.abs() * dw.abs())
    expected = r * (w * (du - inner) + u * dw)
    updated, normalized = (forward_ad.unpack_dual(t).tangent for t in outputs)
    if set(moved) & {"x", "branch"}:
        reference.assert_within(updated, du, reference.U * du.abs(), "updated")
    else:
        assert updated is None
    # u itself, a rounded sum, is u off relative to its terms.
    terms = values["x"].abs() + values["branch"].abs()
    reference.assert_within(normalized, expected,
                            (HIDDEN + 128) * reference.U * size * (terms / u.abs()).amax(),
                            "normalized")


SUBSETS = [s for n in (1, 2, 3) for s in itertools.combinations(PARTS, n)]


@pytest.mark.parametrize("requires_grad", [False, True])
@pytest.mark.parametrize("moved", SUBSETS)
def test_the_pytorch_path_carries_tangents(moved, requires_grad):
    values, directions = make("cpu")
    with forward_ad.dual_level():
        outputs = residual_rms_norm(*dual(values, directions, moved, requires_grad), EPS,
                                    implementation="torch")
        check_tangents(outputs, values, directions, moved)


@pytest.mark.parametrize("part", PARTS)
def test_a_checkpoint_with_a_tangent_is_refused(part):
    values, directions = make("cpu")
    with forward_ad.dual_level(), pytest.raises((RuntimeError, NotImplementedError), match="jvp"):
        residual_rms_norm(*dual(values, directions, [part]), EPS, implementation="torch",
                          checkpoint_dtype=torch.int8)


def check_quantized_refusals(device, implementation):
    values, directions = make(device)
    for part in PARTS:
        with forward_ad.dual_level(), pytest.raises(RuntimeError, match="forward-mode derivative"):
            residual_rms_norm_quantized(*dual(values, directions, [part]), EPS,
                                        implementation=implementation)
    with torch.no_grad():
        _, codes, scale = residual_rms_norm_quantized(*values.values(), EPS,
                                                      implementation=implementation)
    with forward_ad.dual_level(), pytest.raises(RuntimeError, match="forward-mode derivative"):
        dequantize(codes, forward_ad.make_dual(scale, torch.ones_like(scale)),
                   implementation=implementation)


def test_quantized_calls_refuse_tangents():
    check_quantized_refusals("cpu", "torch")


@pytest.mark.gpu
@pytest.mark.parametrize("implementation", ["auto", "gfx950", "torch"])
def test_quantized_calls_refuse_tangents_on_the_gpu(implementation):
    check_quantized_refusals("cuda", implementation)


@pytest.mark.gpu
@pytest.mark.parametrize("requires_grad", [False, True])
@pytest.mark.parametrize("moved", SUBSETS)
def test_auto_takes_the_path_that_carries_tangents(moved, requires_grad):
    values, directions = make("cuda")
    plain = residual_rms_norm(*values.values(), EPS)  # the device is known to be ready
    with forward_ad.dual_level():
        inputs = dual(values, directions, moved, requires_grad)
        assert not can_use_residual_rms_norm(*inputs)
        with pytest.warns(RuntimeWarning, match="forward-mode derivative"):
            outputs = residual_rms_norm(*inputs, EPS)
        check_tangents(outputs, values, directions, moved)
        with pytest.raises(RuntimeError, match="forward-mode derivative"):
            residual_rms_norm(*inputs, EPS, implementation="gfx950")
        # The primals alone are served.
        for a, b in zip(residual_rms_norm(*(forward_ad.unpack_dual(t).primal for t in inputs), EPS,
                                          implementation="gfx950"), plain):
            assert reference.same_bits(a, b)
    for a, b in zip(residual_rms_norm(*values.values(), EPS, implementation="gfx950"), plain):
        assert reference.same_bits(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("checkpoint", [None, torch.int8])
@pytest.mark.parametrize("output", [0, 1])
def test_a_backward_refuses_gradients_with_a_tangent(checkpoint, output):
    values, _ = make("cuda")
    leaves = [t.requires_grad_() for t in values.values()]
    outputs = residual_rms_norm(*leaves, EPS, implementation="gfx950",
                                checkpoint_dtype=checkpoint)
    with forward_ad.dual_level():
        upstream = [torch.ones_like(t) for t in outputs]
        upstream[output] = forward_ad.make_dual(upstream[output], torch.ones_like(outputs[output]))
        with pytest.raises(RuntimeError, match="forward-mode derivative"):
            torch.autograd.grad(outputs, leaves, upstream, retain_graph=True)
    grads = torch.autograd.grad(outputs, leaves, [torch.ones_like(t) for t in outputs])
    assert all(g.isfinite().all() for g in grads)


@pytest.mark.gpu
@pytest.mark.parametrize("part", PARTS)
def test_a_compiled_call_keeps_tangents(part):
    """Tangents made inside of the compiled function, where the custom op would be
    recorded without them."""
    values, directions = make("cuda")

    def derivative(implementation):
        def function(x, branch, weight, direction):
            with forward_ad.dual_level():
                inputs = dict(x=x, branch=branch, weight=weight)
                inputs[part] = forward_ad.make_dual(inputs[part], direction)
                normalized = residual_rms_norm(*inputs.values(), EPS,
                                               implementation=implementation)[1]
                return forward_ad.unpack_dual(normalized).tangent
        return function

    args = [*values.values(), directions[part]]
    torch._dynamo.reset()
    compiled = torch.compile(derivative("auto"), backend="aot_eager", fullgraph=True)(*args)
    torch.testing.assert_close(compiled, derivative("torch")(*args), rtol=1e-5, atol=1e-5)
    torch._dynamo.reset()
    with pytest.raises(Exception, match="forward-mode derivative"):
        torch.compile(derivative("gfx950"), backend="aot_eager")(*args)

    def jvp(implementation):
        return torch.func.jvp(
            lambda t: residual_rms_norm(*(t if k == part else values[k] for k in PARTS), EPS,
                                        implementation=implementation)[1],
            (values[part],), (directions[part],))

    torch._dynamo.reset()
    for a, b in zip(torch.compile(jvp, backend="aot_eager")("auto"), jvp("torch")):
        torch.testing.assert_close(a, b, rtol=1e-5, atol=1e-5)
