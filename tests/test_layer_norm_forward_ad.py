"""Forward-mode derivatives of the residual LayerNorm: carried by the PyTorch path,
which ``"auto"`` takes for inputs with a tangent, and refused by the kernels, which
would drop them."""

import pytest
import torch
from torch.autograd import forward_ad

from gfx1010_kernels import can_use_residual_layer_norm, residual_layer_norm

pytestmark = pytest.mark.gpu
PARTS = ["x", "branch", "weight", "bias"]


def make():
    generator = torch.Generator().manual_seed(0)
    return {k: torch.randn((4, 128) if k in ("x", "branch") else 128, generator=generator).cuda()
            for k in PARTS}


def dual(values, part, requires_grad):
    return [forward_ad.make_dual(v.clone().requires_grad_(requires_grad), torch.ones_like(v))
            if k == part else v for k, v in values.items()]


def tangents(outputs):
    return [forward_ad.unpack_dual(t).tangent for t in outputs]


@pytest.mark.parametrize("requires_grad", [False, True])
@pytest.mark.parametrize("part", PARTS)
def test_auto_takes_the_path_that_carries_tangents(part, requires_grad):
    values = make()
    plain = residual_layer_norm(*values.values(), training=False)
    with forward_ad.dual_level():
        inputs = dual(values, part, requires_grad)
        assert not can_use_residual_layer_norm(*inputs)
        with pytest.warns(RuntimeWarning, match="forward-mode derivative"):
            found = tangents(residual_layer_norm(*inputs, training=False))
        expected = tangents(residual_layer_norm(*inputs, training=False, implementation="torch"))
        assert expected[1] is not None
        for a, b in zip(found, expected):
            assert (a is None and b is None) or torch.equal(a, b)
        with pytest.raises(RuntimeError, match="forward-mode derivative"):
            residual_layer_norm(*inputs, training=False, implementation="gfx950")
    for a, b in zip(residual_layer_norm(*values.values(), training=False), plain):
        assert torch.equal(a, b)


@pytest.mark.parametrize("output", [0, 1])
def test_a_backward_refuses_gradients_with_a_tangent(output):
    leaves = [t.requires_grad_() for t in make().values()]
    outputs = residual_layer_norm(*leaves, training=False)
    with forward_ad.dual_level():
        upstream = [torch.ones_like(t) for t in outputs]
        upstream[output] = forward_ad.make_dual(upstream[output], torch.ones_like(outputs[output]))
        with pytest.raises(RuntimeError, match="forward-mode derivative"):
            torch.autograd.grad(outputs, leaves, upstream, retain_graph=True)
    grads = torch.autograd.grad(outputs, leaves, [torch.ones_like(t) for t in outputs])
    assert all(g.isfinite().all() for g in grads)


@pytest.mark.parametrize("part", PARTS)
def test_a_compiled_call_drops_no_tangent(part):
    """Where the custom op would be recorded without it. PyTorch 2.10 cannot compile
    the forward derivative of its own F.layer_norm and raises; what compiles has to
    carry the tangent."""
    values = make()

    def derivative(implementation):
        def function(*inputs):
            with forward_ad.dual_level():
                inputs = [forward_ad.make_dual(v, torch.ones_like(v)) if k == part else v
                          for k, v in zip(PARTS, inputs)]
                return tangents(residual_layer_norm(*inputs, training=False,
                                                    implementation=implementation))[1]
        return function

    torch._dynamo.reset()
    compiled = torch.compile(derivative("auto"), backend="aot_eager", fullgraph=True)
    try:
        found = compiled(*values.values())
    except torch._dynamo.exc.TorchRuntimeError as error:
        assert "layer_norm" in str(error)
    else:
        torch.testing.assert_close(found, derivative("torch")(*values.values()), rtol=1e-5,
                                   atol=1e-5)
    torch._dynamo.reset()
    with pytest.raises(Exception, match="forward-mode derivative"):
        torch.compile(derivative("gfx950"), backend="aot_eager")(*values.values())
