"""The gated residual norm on the CPU: its reference against differences, the PyTorch
path against the reference, dispatch, and what every entry point refuses."""

import ctypes
import warnings

import pytest
import torch
from torch import nn

import gated_reference as reference
from gfx1010_kernels import (
    _C,
    _cabi,
    can_use_gated_residual_rms_norm,
    gated_norm,
    gated_residual_rms_norm,
    prenorm_forward,
    residual_norm,
    residual_rms_norm,
)

EPS = 1e-6
F64 = torch.float64
KINDS = [(True, "sample", "shared"), (True, "token", "sample"), (False, "shared", "sample"),
         (True, "none", "shared"), (False, "none", "sample"), (True, "sample", "sample")]


def call(parts, **options):
    x, branch, weight, post, gate = parts
    return gated_residual_rms_norm(x, branch, weight, EPS, branch_weight=post, gate=gate,
                                   **options)


@pytest.mark.parametrize("post,gate,weight", KINDS)
def test_torch_path_and_its_gradients_are_the_reference(post, gate, weight):
    parts = reference.make((2, 3, 20), [F64] * 5, post=post, gate=gate, weight=weight, seed=1)
    leaves = [None if t is None else t.requires_grad_() for t in parts]
    options = dict(branch_eps=1e-4, residual_scale=1.25, branch_scale=0.5, implementation="torch")
    updated, normalized = call(leaves, **options)
    call64 = reference.Call(parts, EPS, 1e-4, 1.25, 0.5)
    assert torch.allclose(updated, call64.updated()[0], rtol=0, atol=1e-13)
    upstream = [torch.randn(2, 3, 20, dtype=F64) for _ in range(2)]
    given = [t for t in leaves if t is not None]
    grads = torch.autograd.grad([updated, normalized], given, upstream)
    expected = [e[0] for e in call64.gradients(updated, *upstream) if e is not None]
    for grad, value in zip(grads, expected):
        assert torch.allclose(grad, value, rtol=0, atol=1e-12)

    def outputs(*tensors):
        it = iter(tensors)
        return call([None if t is None else next(it) for t in leaves], **options)

    assert torch.autograd.gradcheck(outputs, given)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_torch_path_in_other_types(dtype):
    parts = reference.make((2, 5, 24), [dtype] * 5, seed=2)
    updated, normalized = call(parts, implementation="torch", normalized_dtype=torch.float32)
    reference.Call(parts, EPS, EPS, 1.0, 1.0).check_forward(updated, normalized, torch.float32,
                                                            dtype)


def test_torch_path_broadcasts_as_torch_does():
    x, branch = torch.randn(2, 3, 4, 8), torch.randn(2, 3, 4, 8)
    gate, weight = torch.randn(3, 1, 8), torch.rand(4, 8)
    updated, normalized = gated_residual_rms_norm(x, branch, weight, gate=gate,
                                                  implementation="torch")
    assert torch.allclose(updated, x + gate * branch)
    rstd = (updated.square().mean(-1, keepdim=True) + EPS).rsqrt()
    assert torch.allclose(normalized, updated * rstd * weight, atol=1e-6)


# Dispatch and refusals.

def test_auto_falls_back_with_a_warning_and_strict_modes_raise():
    parts = reference.make((2, 3, 16), [torch.float32] * 5)
    with pytest.warns(RuntimeWarning, match="gated residual RMSNorm was not used: all tensors must be HIP tensors"):
        call(parts)
    assert not can_use_gated_residual_rms_norm(*parts[:3])
    for implementation in ("gfx950", "gfx1010"):
        with pytest.raises(RuntimeError, match="must be HIP tensors"):
            call(parts, implementation=implementation)
    with pytest.raises(RuntimeError, match="Triton backend"):
        call(parts, implementation="triton")
    with pytest.raises(ValueError, match="implementation must be"):
        call(parts, implementation="hip")
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        call(parts, implementation="torch")


@pytest.mark.parametrize("changes,message", [
    (dict(normalized_dtype=F64), "normalized_dtype"),
    (dict(branch=torch.zeros(2, 16)), "same shape"),
    (dict(branch_weight=torch.zeros(8)), "branch_weight must match"),
    (dict(branch_weight=torch.zeros(1, 16)), "branch_weight must match"),
    (dict(weight=torch.zeros(8)), "weight must match"),
    (dict(weight=torch.zeros(())), "weight must match"),
    (dict(gate=torch.zeros(3, 1, 16)), "gate must match"),
    (dict(gate=torch.zeros(2, 3, 1)), "gate must match"),
    (dict(gate=torch.zeros(1, 2, 3, 16)), "gate must match"),
])
def test_argument_checks(changes, message):
    args = dict(x=torch.zeros(2, 3, 16), branch=torch.zeros(2, 3, 16), weight=torch.ones(16))
    for implementation in ("auto", "torch"):
        with pytest.raises(ValueError, match=message):
            gated_residual_rms_norm(**dict(args, **changes), implementation=implementation)


class Device:
    """A tensor's attributes as a HIP tensor has them."""

    def __init__(self, shape, dtype=torch.float32, device=0):
        self.is_cuda, self.device = True, torch.device("cuda", device)
        self.shape, self.ndim, self.dtype = torch.Size(shape), len(shape), dtype

    def numel(self):
        return self.shape.numel()


def reason(x=(4, 6, 32), branch=None, weight=(32,), post=None, gate=None, eps=EPS, branch_eps=EPS,
           scales=(1.0, 1.0)):
    def made(given):
        return given if given is None or isinstance(given, Device) else Device(given)

    x = made(x)
    return gated_norm._input_reason(x, made(branch or x.shape), made(weight), made(post),
                                    made(gate), eps, branch_eps, *scales)


def test_reasons():
    for gate in (None, (32,), (1, 32), (1, 1, 32), (4, 1, 32), (4, 6, 32)):
        assert reason(gate=gate, post=(32,)) is None
        assert reason(gate=gate, weight=(4, 1, 32)) is None
    assert reason(x=(4, 2, 3, 32), gate=(4, 2, 1, 32)) is None
    assert reason(x=(0, 6, 32), gate=(0, 1, 32)) is None
    assert reason(x=(32,)) is None
    assert reason(x=(4, 2, 3, 32), gate=(4, 2, 3, 32), weight=(4, 1, 1, 32)) is None
    for text, changes in [
        ("same HIP device", dict(weight=Device((32,), device=1))),
        ("must use float16", dict(gate=Device((32,), F64))),
        ("same shape", dict(branch=(4, 32))),
        ("hidden size", dict(x=(4, 0))),
        ("hidden size", dict(x=(4, 16385))),
        ("branch_weight must match", dict(post=(31,))),
        ("must repeat over the last", dict(gate=(6, 32))),
        ("must repeat over the last", dict(gate=(1, 6, 32))),
        ("must repeat over the last", dict(weight=(4, 6, 1))),
        ("same rows", dict(x=(4, 2, 3, 32), gate=(4, 1, 1, 32), weight=(4, 2, 1, 32))),
        ("same rows", dict(gate=(4, 1, 32), weight=(4, 6, 32))),
        ("eps", dict(eps=-1.0)),
        ("eps", dict(branch_eps=float("nan"))),
        ("finite", dict(scales=(float("inf"), 1.0))),
    ]:
        assert text in reason(**changes), changes


def test_the_extension_declines_host_tensors():
    x, branch, weight, post, gate = reference.make((2, 3, 16), [torch.float32] * 5)
    args = (x, branch, weight, post, gate, EPS, EPS, 1.0, 1.0)
    assert _C.gated_residual_rms_norm_if_supported(*args, None) is None
    assert _C.gated_inputs_refusal(*args) == "all tensors must be HIP tensors"
    for function in (_C.gated_residual_rms_norm, _C.gated_residual_rms_norm_forward):
        with pytest.raises(RuntimeError, match="must be HIP tensors"):
            function(*args, None)
    with pytest.raises(RuntimeError, match="must be HIP tensors"):
        _C.gated_residual_rms_norm_backward(x, x, x, branch, weight, post, gate, x, 1.0, 1.0, 31)


# The C ABI.

FAKE = 1 << 20  # a non-null address; validation fails before it is touched
F32, F16, BF16, INT8 = range(4)


def factor(data=FAKE, dtype=BF16, stride=768, rows=4):
    return ctypes.byref(_cabi.RlnFactor(data, dtype, stride, rows))


def check(status, message):
    assert status != 0 and message in _cabi.last_error(), (status, _cabi.last_error())


COMMON = [
    (dict(rows=0), "empty tensors"),
    (dict(hidden=0), "hidden size: 0"),
    (dict(hidden=16385), "hidden size: 16385"),
    (dict(rows=1 << 60), "overflows"),
    (dict(branch=None), "must not be null"),
    (dict(weight=None), "must not be null"),
    (dict(weight=factor(data=None)), "must not be null"),
    (dict(x_dtype=INT8), "x must use"),
    (dict(branch_dtype=7), "branch must use"),
    (dict(branch_weight_dtype=-1), "branch_weight must use"),
    (dict(gate=factor(dtype=INT8)), "gate must use"),
    (dict(weight=factor(dtype=9)), "weight must use"),
    (dict(gate=factor(rows=3)), "gate: its rows"),
    (dict(gate=factor(rows=0)), "gate: its rows"),
    (dict(weight=factor(rows=-4)), "weight: its rows"),
    (dict(gate=factor(rows=2), weight=factor(rows=1)), "same rows"),
    (dict(gate=factor(data=FAKE + 1)), "gate is not aligned"),
    (dict(branch=FAKE + 1), "branch is not aligned"),
    (dict(branch_stride=1 << 61), "branch: the row stride overflows"),
    (dict(weight=factor(stride=-(1 << 62), rows=2)), "weight: the row stride overflows"),
    (dict(residual_scale=float("nan")), "must be finite"),
    (dict(branch_scale=float("inf")), "must be finite"),
]


@pytest.mark.parametrize("changes,message", COMMON + [
    (dict(x=None), "must not be null"),
    (dict(updated=None), "must not be null"),
    (dict(normalized=None), "must not be null"),
    (dict(normalized_dtype=INT8), "normalized must use"),
    (dict(normalized=FAKE + 1), "normalized is not aligned"),
    (dict(x_stride=-(1 << 61)), "x: the row stride overflows"),
    (dict(statistics=FAKE + 2), "statistics is not aligned"),
    (dict(eps=-1.0), "eps"),
    (dict(branch_eps=float("nan")), "eps"),
])
def test_forward_refusals(changes, message):
    args = dict(x=FAKE, x_dtype=BF16, x_stride=768, branch=FAKE, branch_dtype=BF16,
                branch_stride=768, branch_weight=FAKE, branch_weight_dtype=BF16, gate=factor(),
                weight=factor(), updated=FAKE, normalized=FAKE, normalized_dtype=BF16,
                statistics=None, rows=4, hidden=768, residual_scale=1.0, branch_scale=1.0,
                eps=EPS, branch_eps=EPS, stream=None)
    check(_cabi.library().rln_gated_forward(*dict(args, **changes).values()), message)


@pytest.mark.parametrize("changes,message", COMMON + [
    (dict(updated=None), "must not be null"),
    (dict(statistics=None), "must not be null"),
    (dict(grad_x=None), "must not be null"),
    (dict(grad_branch=None), "must not be null"),
    (dict(gate=None, grad_gate=FAKE), "without a gate"),
    (dict(branch_weight=None, grad_branch_weight=FAKE), "without a branch_weight"),
    (dict(grad_normalized_dtype=INT8), "grad_normalized must use"),
    (dict(grad_updated=FAKE + 1), "grad_updated is not aligned"),
    (dict(grad_gate=FAKE + 1), "grad_gate is not aligned"),
    (dict(grad_weight=FAKE), "workspace too small"),
    (dict(grad_gate=FAKE, workspace=FAKE, workspace_bytes=16), "workspace too small"),
    (dict(workspace=FAKE + 2), "workspace is not aligned"),
])
def test_backward_refusals(changes, message):
    args = dict(grad_updated=FAKE, grad_normalized=FAKE, grad_normalized_dtype=BF16, updated=FAKE,
                x_dtype=BF16, branch=FAKE, branch_dtype=BF16, branch_stride=768,
                branch_weight=FAKE, branch_weight_dtype=BF16, gate=factor(), weight=factor(),
                statistics=FAKE, grad_x=FAKE, grad_branch=FAKE, grad_gate=None,
                grad_branch_weight=None, grad_weight=None, rows=4, hidden=768,
                residual_scale=1.0, branch_scale=1.0, workspace=None, workspace_bytes=0,
                stream=None)
    check(_cabi.library().rln_gated_backward(*dict(args, **changes).values()), message)


def test_workspace_sizes():
    size = _cabi.library().rln_gated_backward_workspace_bytes
    for rows in (1, 6, 1000, 1 << 20, (1 << 40) + 8):
        for hidden in (1, 64, 768, 4097, 16384):
            for dtype in (F32, F16, BF16):
                shared = size(rows, hidden, dtype, rows, rows)
                assert 8 * hidden <= shared <= 512 * 8 * hidden
                # token gates have more units, and other groups a sum each at least
                assert shared <= size(rows, hidden, dtype, 1, rows) <= 512 * 8 * hidden
                if rows % 2 == 0:
                    assert size(rows, hidden, dtype, 2, rows) >= rows // 2 * 8 * hidden
                    assert size(rows, hidden, dtype, rows // 2, rows) >= 16 * hidden
    for bad in ((0, 64, F32, 1, 1), (4, 0, F32, 4, 4), (4, 64, INT8, 4, 4), (4, 64, F32, 3, 4),
                (4, 64, F32, 0, 4), (4, 64, F32, 4, -4), (-8, 64, F32, 4, 4)):
        assert size(*bad) == 0


@pytest.mark.parametrize("post", [True, False])
def test_fake_shapes(post):
    from torch._subclasses.fake_tensor import FakeTensorMode

    ops = torch.ops.gfx1010_kernels
    with FakeTensorMode():
        x = torch.empty(2, 3, 40, device="cuda", dtype=torch.bfloat16)
        branch = torch.empty(2, 3, 40, device="cuda")
        weight = torch.empty(40, device="cuda")
        gate = torch.empty(2, 1, 40, device="cuda", dtype=torch.float16)
        own = torch.empty(40, device="cuda") if post else None
        updated, normalized, statistics = ops.gated_forward(x, branch, weight, own, gate, EPS, EPS,
                                                            1.0, 1.0, torch.float16)
        assert updated.shape == x.shape and updated.dtype == x.dtype
        assert normalized.shape == x.shape and normalized.dtype == torch.float16
        assert statistics.shape == (12 if post else 6,) and statistics.dtype == torch.float32
        grads = ops.gated_backward(updated, normalized, updated, branch, weight, own, gate,
                                   statistics, 1.0, 1.0, 31)
        for grad, part in zip(grads, (x, branch, weight, own, gate)):
            if part is None:
                assert grad.shape == (0,)
            else:
                assert grad.shape == part.shape and grad.dtype == part.dtype


# The pre-norm helpers.

class SandwichBlock(nn.Module):
    def __init__(self, hidden):
        super().__init__()
        self.ln_1, self.post_1 = nn.RMSNorm(hidden, eps=1e-5), nn.RMSNorm(hidden, eps=1e-4)
        self.ln_2, self.post_2 = nn.RMSNorm(hidden, eps=1e-5), nn.RMSNorm(hidden)
        self.attn = nn.Linear(hidden, hidden)
        self.mlp = nn.Sequential(nn.Linear(hidden, 2 * hidden), nn.SiLU(),
                                 nn.Linear(2 * hidden, hidden))
        self.gate = nn.Parameter(torch.randn(hidden))


@pytest.mark.parametrize("posts", [True, False])
@pytest.mark.parametrize("gates", [True, False])
def test_prenorm_stack_of_gated_blocks(posts, gates):
    torch.manual_seed(3)
    blocks = nn.ModuleList(SandwichBlock(32) for _ in range(3)).double()
    final = nn.RMSNorm(32).double()
    x = torch.randn(2, 5, 32, dtype=F64)
    options = dict(residual_scale=1.0 if posts else 0.9, branch_scale=0.7)
    if posts:
        options.update(post_ln1="post_1", post_ln2=lambda block: block.post_2)
    if gates:
        options.update(gate1="gate", gate2=lambda block: block.gate.tanh())
    with warnings.catch_warnings():
        warnings.simplefilter("ignore")
        stream, out = prenorm_forward(x, blocks, final, **options)
    expected = x
    for block in blocks:
        added = block.attn(block.ln_1(expected))
        added = block.post_1(added) if posts else added
        added = added * block.gate if gates else added
        expected = options["residual_scale"] * expected + 0.7 * added
        added = block.mlp(block.ln_2(expected))
        added = block.post_2(added) if posts else added
        added = added * block.gate.tanh() if gates else added
        expected = options["residual_scale"] * expected + 0.7 * added
    assert torch.allclose(stream, expected, atol=1e-9)
    # A module without an eps adds fp32's.
    eps = torch.finfo(torch.float32).eps
    value = expected * (expected.square().mean(-1, keepdim=True) + eps).rsqrt() * final.weight
    assert torch.allclose(out, value, atol=1e-6)


def test_residual_norm_refuses_what_it_cannot_fuse():
    x = torch.randn(2, 16)
    layer, rms = nn.LayerNorm(16), nn.RMSNorm(16)
    for options in (dict(gate=torch.ones(16)), dict(branch_norm=rms), dict(branch_scale=0.5)):
        with pytest.raises(TypeError, match="RMSNorm"):
            residual_norm(x, x, layer, **options)
    with pytest.raises(TypeError, match="RMSNorm"):
        residual_norm(x, x, rms, branch_norm=layer)
    with pytest.raises(ValueError, match="hidden size"):
        residual_norm(x, x, rms, branch_norm=nn.RMSNorm(8))
    with pytest.raises(ValueError, match="checkpoint_dtype"):
        residual_norm(x, x, rms, gate=torch.ones(16), checkpoint_dtype=torch.int8)


def test_without_gate_and_weight_it_is_the_residual_norm():
    x, branch, weight = torch.randn(3, 40), torch.randn(3, 40), torch.rand(40)
    options = dict(implementation="torch")
    for a, b in zip(gated_residual_rms_norm(x, branch, weight, EPS, **options),
                    residual_rms_norm(x, branch, weight, EPS, **options)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("value", [1.0, 0.5])
@pytest.mark.parametrize("which", ["residual_scale", "branch_scale"])
def test_scales_lose_no_gradient(which, value):
    """A scale is a number; a tensor that requires a gradient is refused, whatever it holds."""
    import numpy as np

    x, branch, weight, _, _ = reference.make((2, 3, 8), [torch.float32] * 5)
    scale = {which: torch.nn.Parameter(torch.tensor(value))}
    norm = torch.nn.RMSNorm(8, eps=1e-6)
    for implementation in ("auto", "torch", "gfx950"):
        with pytest.raises(ValueError, match=f"{which} is a number"):
            gated_residual_rms_norm(x, branch, weight, **scale, implementation=implementation)
        with pytest.raises(ValueError, match=f"{which} is a number"):
            residual_norm(x, branch, norm, **scale, implementation=implementation)
    number = {which: value}
    for given in (scale, {which: torch.tensor(value)}, {which: np.float32(value)}):
        with torch.no_grad():
            for a, b in zip(gated_residual_rms_norm(x, branch, weight, **given,
                                                    implementation="torch"),
                            gated_residual_rms_norm(x, branch, weight, **number,
                                                    implementation="torch")):
                assert torch.equal(a, b)
