"""The root-mean-square norm operators on the CPU: the PyTorch path against the
64-bit reference, the reference's gradients against differences, the dispatch,
the C ABI's refusals (no GPU work: every call fails its checks first), the
custom ops' shapes and the pre-norm helpers with ``nn.RMSNorm``.
"""

import warnings

import pytest
import torch
from torch import nn
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.nn import functional as F

import rms_reference as reference
from gfx1010_kernels import (
    _cabi,
    can_use_residual_rms_norm,
    dequantize,
    prenorm_forward,
    residual_norm,
    residual_rms_norm,
    residual_rms_norm_quantized,
    rms_norm,
)

EPS = 1e-6
CODES = [torch.int8, torch.float8_e4m3fn]
GROUPS = [None, 32, 64, 128, 256]


def make(shape, x_dtype=torch.float32, branch_dtype=torch.float32, weight_dtype=torch.float32,
         seed=0):
    generator = torch.Generator().manual_seed(seed)
    x = (2.0 * torch.randn(shape, generator=generator)).to(x_dtype)
    branch = torch.randn(shape, generator=generator).to(branch_dtype)
    weight = (1.0 + 0.1 * torch.randn(shape[-1], generator=generator)).to(weight_dtype)
    return x, branch, weight


# The 64-bit reference itself.

@pytest.mark.parametrize("hidden", [1, 5, 64])
def test_reference_gradients_are_those_of_autograd_and_of_differences(hidden):
    x, _, weight = (t.double() for t in make((3, hidden)))
    grad_updated, grad_normalized = torch.randn(3, hidden).double(), torch.randn(3, hidden).double()
    leaves = [x.requires_grad_(), weight.requires_grad_()]

    def loss(u, w):
        return (u * grad_updated).sum() + (reference.normalized(u, w, EPS) * grad_normalized).sum()

    expected = torch.autograd.grad(loss(*leaves), leaves)
    g, grad_weight, _, _ = reference.gradients(x.detach(), x.detach(), weight.detach(), EPS,
                                               grad_updated, grad_normalized)
    torch.testing.assert_close(g, expected[0], rtol=1e-12, atol=1e-12)
    torch.testing.assert_close(grad_weight, expected[1], rtol=1e-12, atol=1e-12)
    h = 1e-6
    with torch.no_grad():
        for row, column in [(0, 0), (2, hidden - 1)]:
            step = torch.zeros_like(x)
            step[row, column] = h
            slope = (loss(x + step, weight) - loss(x - step, weight)) / (2 * h)
            assert abs(slope - g[row, column]) < 1e-6 * (1 + abs(slope))


# The PyTorch path.

@pytest.mark.parametrize("dtypes", [(torch.float32,) * 3, (torch.bfloat16,) * 3,
                                    (torch.float32, torch.float16, torch.float32)])
@pytest.mark.parametrize("shape", [(4,), (3, 7), (2, 5, 129), (0, 16), (2, 0, 16)])
def test_torch_path_matches_the_reference(shape, dtypes):
    x, branch, weight = make(shape, *dtypes)
    for added in (branch, None):
        updated, normalized = residual_rms_norm(x, added, weight, EPS, implementation="torch")
        expected = reference.update(x, added)
        assert torch.equal(updated, expected) and normalized.dtype == x.dtype
        value = reference.normalized(expected, weight, EPS)
        reference.assert_within(normalized, value,
                                reference.normalized_bound(value, x.dtype), "normalized")
    assert residual_rms_norm(x, None, weight, implementation="torch")[0] is x


@pytest.mark.parametrize("dtype", CODES)
@pytest.mark.parametrize("group", GROUPS)
@pytest.mark.parametrize("hidden", [1, 31, 100, 256, 300])
def test_torch_path_quantizes_as_defined(hidden, group, dtype):
    x, branch, weight = make((5, hidden), torch.bfloat16, torch.bfloat16, torch.bfloat16)
    x[3] = 0
    branch[3] = 0
    updated, codes, scale = residual_rms_norm_quantized(
        x, branch, weight, EPS, dtype=dtype, group_size=group, implementation="torch")
    expected_codes, expected_scale = reference.quantized(updated, weight, EPS, group, dtype)
    assert reference.same_bits(codes, expected_codes)
    assert scale.shape == expected_scale.shape and scale.dtype == torch.float32
    torch.testing.assert_close(scale.double(), expected_scale, rtol=1e-5, atol=0)
    assert not codes[3].float().any()
    values = dequantize(codes, scale, group_size=group, dtype=torch.float32,
                        implementation="torch")
    wide = reference.normalized(updated, weight, EPS)
    # Half a step of the group's scale, e4m3's own step near its largest value.
    half = {torch.int8: 0.5, torch.float8_e4m3fn: 16.0}[dtype]
    steps = reference.spread(expected_scale, group or hidden, hidden)
    assert ((values.double() - wide).abs() <= half * 1.0001 * steps + 1e-30).all()


@pytest.mark.parametrize("hidden", [5, 200])
def test_torch_path_keeps_fp64(hidden):
    """fp64 tensors, which the kernels do not take, are computed in fp64."""
    x, branch, weight = (t.double() for t in make((4, hidden)))
    branch = branch + 2.0 ** -40
    updated, normalized = residual_rms_norm(x, branch, weight, EPS, implementation="torch")
    assert torch.equal(updated, x + branch) and normalized.dtype == torch.float64
    torch.testing.assert_close(normalized, F.rms_norm(x + branch, (hidden,), weight, EPS),
                               rtol=1e-14, atol=1e-14)
    assert torch.autograd.gradcheck(
        lambda *t: residual_rms_norm(*t, EPS, implementation="torch"),
        [t.requires_grad_() for t in (x, branch, weight)], atol=1e-6)
    with torch.no_grad():
        _, codes, scale = residual_rms_norm_quantized(x, branch, weight, EPS,
                                                      implementation="torch")
    assert scale.dtype == torch.float32
    assert (dequantize(codes, scale, dtype=torch.float32, implementation="torch") - normalized
            ).abs().max() <= 16.001 * scale.max()


def test_torch_path_marks_groups_that_are_not_finite():
    x = torch.randn(2, 256)
    x[0, 130] = float("inf")
    x[1, 5] = float("nan")
    _, codes, scale = residual_rms_norm_quantized(
        x, None, torch.ones(256), dtype=torch.int8, group_size=128, implementation="torch")
    assert scale[0, 0] == 0 and scale[0, 1].isnan() and scale[1].isnan().all()
    values = dequantize(codes, scale, group_size=128, implementation="torch")
    assert (values[0, :128] == 0).all() and values[0, 128:].isnan().all()


@pytest.mark.parametrize("hidden", [1, 100, 384])
def test_torch_checkpoint_gradients(hidden):
    x, branch, weight = make((6, hidden))
    leaves = [t.requires_grad_() for t in (x, branch, weight)]
    updated, normalized = residual_rms_norm(*leaves, EPS, implementation="torch",
                                            checkpoint_dtype=torch.int8)
    grads = [torch.randn_like(updated), torch.randn_like(updated)]
    grad_x, grad_branch, grad_weight = torch.autograd.grad([updated, normalized], leaves, grads)
    u = updated.detach()
    g, gw, size, terms = reference.gradients(u, reference.checkpoint(u)[2], weight.detach(), EPS,
                                             *grads)
    # torch's own sums: at most `hidden` or 6 additions.
    bound = reference.rounding(g, (128 + hidden) * reference.U * size, torch.float32)
    reference.assert_within(grad_x, g, bound, "grad_x")
    assert torch.equal(grad_x, grad_branch)
    reference.assert_within(grad_weight, gw,
                            reference.weight_bound(gw, terms, hidden, torch.float32), "weight")


# Dispatch.

def test_auto_falls_back_with_a_warning_and_strict_modes_raise():
    x, branch, weight = make((2, 16))
    with pytest.warns(RuntimeWarning, match="was not used: x, branch and weight must be HIP"):
        updated, normalized = residual_rms_norm(x, branch, weight)
    assert torch.equal(updated, x + branch)
    torch.testing.assert_close(normalized, F.rms_norm(x + branch, (16,), weight, 1e-6))
    with pytest.warns(RuntimeWarning, match="was not used"):
        codes, scale = residual_rms_norm_quantized(x, branch, weight)[1:]
    with pytest.warns(RuntimeWarning, match="was not used"):
        dequantize(codes, scale)
    assert not can_use_residual_rms_norm(x, branch, weight)
    for implementation in ("gfx950", "gfx1010"):
        with pytest.raises(RuntimeError, match="must be HIP tensors"):
            residual_rms_norm(x, branch, weight, implementation=implementation)
        with pytest.raises(RuntimeError, match="must be HIP tensors"):
            residual_rms_norm_quantized(x, branch, weight, implementation=implementation)
        with pytest.raises(RuntimeError, match="must be HIP tensors"):
            dequantize(codes, scale, implementation=implementation)
    with pytest.raises(RuntimeError, match="Triton backend"):
        residual_rms_norm(x, branch, weight, implementation="triton")


def test_argument_checks():
    x, branch, weight = make((2, 64))
    with pytest.raises(ValueError, match="implementation must be"):
        residual_rms_norm(x, branch, weight, implementation="hip")
    with pytest.raises(ValueError, match="normalized_dtype"):
        residual_rms_norm(x, branch, weight, normalized_dtype=torch.float64)
    with pytest.raises(ValueError, match="checkpoint_dtype"):
        residual_rms_norm(x, branch, weight, checkpoint_dtype=torch.float8_e4m3fn)
    with pytest.raises(ValueError, match="dtype must be"):
        residual_rms_norm_quantized(x, branch, weight, dtype=torch.uint8)
    with pytest.raises(ValueError, match="group_size"):
        residual_rms_norm_quantized(x, branch, weight, group_size=48)
    with pytest.raises(RuntimeError, match="records no gradient"):
        residual_rms_norm_quantized(x, branch, weight.clone().requires_grad_())
    codes, scale = torch.zeros(2, 64, dtype=torch.int8), torch.ones(2, 1)
    for bad in (dict(group_size=32), dict(dtype=torch.float64), dict(group_size=7)):
        with pytest.raises(ValueError):
            dequantize(codes, scale, **bad)
    with pytest.raises(ValueError, match="quantized must use"):
        dequantize(codes.float(), scale)
    with pytest.raises(ValueError, match="scale must use"):
        dequantize(codes, scale.half())
    with pytest.raises(ValueError, match="scale must have shape"):
        dequantize(codes, torch.ones(2))


def test_reasons():
    x, branch, weight = make((2, 64))

    class Device:
        """A tensor's attributes as a HIP tensor has them."""

        def __init__(self, tensor, **changes):
            self.is_cuda, self.device = True, torch.device("cuda", 0)
            self.ndim, self.shape, self.dtype = tensor.ndim, tensor.shape, tensor.dtype
            self.__dict__.update(changes)

    good = Device(x), Device(branch), Device(weight)
    assert rms_norm._input_reason(*good, EPS) is None
    assert rms_norm._input_reason(good[0], None, good[2], 0.0) is None
    cases = [
        ((good[0], good[1], Device(weight, device=torch.device("cuda", 1))), EPS, "same device"),
        ((good[0], Device(branch, shape=torch.Size((2, 32))), good[2]), EPS, "same shape"),
        ((Device(x, shape=torch.Size((2, 0))), None, good[2]), EPS, "hidden size"),
        ((Device(x, shape=torch.Size((2, 16385))), None, good[2]), EPS, "hidden size"),
        ((good[0], good[1], Device(weight, shape=torch.Size((63,)))), EPS, "weight must match"),
        ((Device(x, dtype=torch.float64), good[1], good[2]), EPS, "must use float16"),
        (good, -1.0, "eps"),
        (good, float("nan"), "eps"),
    ]
    for tensors, eps, reason in cases:
        assert reason in rms_norm._input_reason(*tensors, eps)


# The C ABI.

FAKE = 1 << 20  # a non-null address; validation fails before it is touched
F32, F16, BF16, INT8, E4M3 = range(5)


def _forward(**changes):
    args = dict(x=FAKE, x_dtype=BF16, weight=FAKE, weight_dtype=BF16, normalized=FAKE,
                normalized_dtype=BF16, rows=4, hidden=768, eps=EPS, branch=FAKE,
                branch_dtype=BF16, updated=FAKE)
    _cabi.rms_forward(**dict(args, **changes))


def _quantize(**changes):
    args = dict(x=FAKE, x_dtype=BF16, weight=FAKE, weight_dtype=BF16, quantized=FAKE,
                quantized_dtype=INT8, scale=FAKE, group=0, rows=4, hidden=768, eps=EPS,
                branch=FAKE, branch_dtype=BF16, updated=FAKE)
    _cabi.rms_quantize(**dict(args, **changes))


SHARED = [
    (dict(rows=0), "empty tensors are unsupported"),
    (dict(hidden=0), "unsupported RMSNorm hidden size: 0"),
    (dict(hidden=16385), "unsupported RMSNorm hidden size: 16385"),
    (dict(rows=1 << 60), "overflows"),
    (dict(x=None), "must not be null"),
    (dict(weight=None), "must not be null"),
    (dict(x_dtype=INT8), "x must use"),
    (dict(branch_dtype=7), "branch must use"),
    (dict(weight_dtype=-1), "weight must use"),
    (dict(branch=None), "both be given or both be null"),
    (dict(updated=None), "both be given or both be null"),
    (dict(eps=-1.0), "eps must not be negative"),
    (dict(eps=float("nan")), "eps must not be negative"),
    (dict(x_stride=1 << 61), "x: the row stride overflows"),
    (dict(branch_stride=-(1 << 61)), "branch: the row stride overflows"),
    (dict(x=FAKE + 1), "x is not aligned"),
    (dict(branch=FAKE + 1), "branch is not aligned"),
    (dict(weight=FAKE + 2, weight_dtype=F32), "weight is not aligned"),
    (dict(updated=FAKE + 1), "updated is not aligned"),
]


@pytest.mark.parametrize("changes,message", SHARED + [
    (dict(normalized=None), "must not be null"),
    (dict(normalized_dtype=E4M3), "normalized must use"),
    (dict(normalized=FAKE + 1), "normalized is not aligned"),
    (dict(rstd=FAKE + 2), "rstd is not aligned"),
    (dict(checkpoint=FAKE, checkpoint_scale=FAKE + 1), "checkpoint_scale is not aligned"),
    (dict(checkpoint=FAKE), "checkpoint and checkpoint_scale must both"),
])
def test_forward_refusals(changes, message):
    with pytest.raises(_cabi.RlnError, match=message):
        _forward(**changes)


@pytest.mark.parametrize("changes,message", SHARED + [
    (dict(quantized=None), "must not be null"),
    (dict(scale=None), "must not be null"),
    (dict(quantized_dtype=BF16), "quantized must use"),
    (dict(group=48), "group must be"),
    (dict(group=-32), "group must be"),
    (dict(scale=FAKE + 1), "scale is not aligned"),
])
def test_quantize_refusals(changes, message):
    with pytest.raises(_cabi.RlnError, match=message):
        _quantize(**changes)


@pytest.mark.parametrize("changes,message", [
    (dict(rows=-1), "empty tensors are unsupported"),
    (dict(hidden=20000), "unsupported RMSNorm hidden size"),
    (dict(x_dtype=9), "x must use"),
    (dict(grad_normalized_dtype=INT8), "grad_normalized must use"),
    (dict(weight_dtype=INT8), "weight must use"),
    (dict(grad_branch=FAKE, branch_dtype=INT8), "branch must use"),
    (dict(grad_normalized=None), "must not be null"),
    (dict(weight=None), "must not be null"),
    (dict(rstd=None), "must not be null"),
    (dict(grad_x=None), "must not be null"),
    (dict(updated=None), "either updated or checkpoint"),
    (dict(checkpoint=FAKE, checkpoint_scale=FAKE), "either updated or checkpoint"),
    (dict(updated=None, checkpoint=FAKE), "either updated or checkpoint"),
    (dict(grad_updated=FAKE + 1), "grad_updated is not aligned"),
    (dict(rows=1 << 16, grad_weight=FAKE), "workspace too small"),
    (dict(rows=1 << 16, grad_weight=FAKE, workspace=FAKE, workspace_bytes=8),
     "workspace too small"),
    (dict(workspace=FAKE + 2), "workspace is not aligned"),
    (dict(rstd=FAKE + 1), "rstd is not aligned"),
    (dict(updated=None, checkpoint=FAKE, checkpoint_scale=FAKE + 3),
     "checkpoint_scale is not aligned"),
    (dict(updated_stride=1 << 61), "updated: the row stride overflows"),
])
def test_backward_refusals(changes, message):
    args = dict(grad_updated=FAKE, grad_normalized=FAKE, grad_normalized_dtype=BF16, x_dtype=BF16,
                weight=FAKE, weight_dtype=BF16, rstd=FAKE, grad_x=FAKE, rows=4, hidden=768,
                updated=FAKE)
    with pytest.raises(_cabi.RlnError, match=message):
        _cabi.rms_backward(**dict(args, **changes))


@pytest.mark.parametrize("changes,message", [
    (dict(rows=0), "empty tensors are unsupported"),
    (dict(hidden=0), "empty tensors are unsupported"),
    (dict(hidden=1 << 31), "unsupported row length"),
    (dict(rows=1 << 60), "overflows"),
    (dict(quantized_dtype=F16), "quantized must use"),
    (dict(values_dtype=INT8), "values must use"),
    (dict(group=16), "group must be"),
    (dict(quantized=None), "must not be null"),
    (dict(scale=None), "must not be null"),
    (dict(values=None), "must not be null"),
    (dict(scale=FAKE + 2), "scale is not aligned"),
    (dict(values=FAKE + 1), "values is not aligned"),
])
def test_dequantize_refusals(changes, message):
    args = dict(quantized=FAKE, quantized_dtype=INT8, scale=FAKE, group=0, values=FAKE,
                values_dtype=BF16, rows=4, hidden=768)
    with pytest.raises(_cabi.RlnError, match=message):
        _cabi.dequantize(**dict(args, **changes))


def test_size_queries():
    library = _cabi.library()
    for hidden, served in [(0, 0), (1, 1), (129, 1), (16384, 1), (16385, 0), (-5, 0)]:
        assert library.rln_rms_hidden_supported(hidden) == served
    assert _cabi.rms_backward_workspace_bytes(0, 768, BF16) == 0
    assert _cabi.rms_backward_workspace_bytes(8, 20000, BF16) == 0
    assert _cabi.rms_backward_workspace_bytes(8, 768, INT8) == 0
    for dtype in (F32, F16, BF16):
        for hidden in (1, 768, 16384):
            few, many = (_cabi.rms_backward_workspace_bytes(rows, hidden, dtype)
                         for rows in (1, 1 << 24))
            # Small launches take none; others a row of sums per block, bounded
            # however many rows there are.
            assert few == 0 and many > 0 and many % (4 * hidden) == 0
            assert many // (4 * hidden) <= 512


def test_glue_declines_host_tensors():
    from gfx1010_kernels import _C

    x, branch, weight = make((2, 64))
    assert _C.rms_inputs_supported(x, branch, weight, EPS) is False
    assert _C.residual_rms_norm_if_supported(x, None, weight, EPS, None, False) is None
    for call in (lambda: _C.residual_rms_norm(x, branch, weight, EPS, None, False),
                 lambda: _C.residual_rms_norm_forward(x, None, weight, EPS, None, True),
                 lambda: _C.residual_rms_norm_quantized(x, branch, weight, EPS, torch.int8, 0)):
        with pytest.raises(RuntimeError, match="x must be a HIP tensor"):
            call()
    with pytest.raises(RuntimeError, match="quantized must be a HIP tensor"):
        _C.dequantize(torch.zeros(2, 4, dtype=torch.int8), torch.ones(2, 1), 0, torch.float32)


# torch.library.

@pytest.mark.parametrize("checkpoint", [False, True])
@pytest.mark.parametrize("shape", [(7, 128), (2, 5, 130), (4,)])
def test_fake_shapes(shape, checkpoint):
    ops = torch.ops.gfx1010_kernels
    hidden, rows = shape[-1], torch.Size(shape).numel() // shape[-1]
    with FakeTensorMode():
        x = torch.empty(shape, device="cuda", dtype=torch.bfloat16)
        branch = torch.empty(shape, device="cuda")
        weight = torch.empty(hidden, device="cuda")
        updated, normalized, state = ops.rms_forward(x, branch, weight, EPS, torch.float16,
                                                     checkpoint)
        assert updated.shape == x.shape and updated.dtype == torch.bfloat16
        assert normalized.shape == x.shape and normalized.dtype == torch.float16
        assert state.dtype == torch.uint8 and state.numel() >= 4 * rows
        grads = ops.rms_backward(updated, normalized, None if checkpoint else updated, state,
                                 weight, torch.bfloat16, torch.float32, checkpoint, True)
        assert grads[0].shape == x.shape and grads[0].dtype == torch.bfloat16
        assert grads[1].shape == x.shape and grads[1].dtype == torch.float32
        assert grads[2].shape == weight.shape
        _, codes, scale = ops.rms_quantized(x, None, weight, EPS, torch.int8, 128)
        assert codes.shape == x.shape and codes.dtype == torch.int8
        assert scale.shape == (*shape[:-1], -(-hidden // 128)) and scale.dtype == torch.float32
        values = ops.dequantize(codes, scale, 128, torch.float16)
        assert values.shape == x.shape and values.dtype == torch.float16


# The pre-norm helpers.

class RmsBlock(nn.Module):
    def __init__(self, hidden):
        super().__init__()
        self.ln_1 = nn.RMSNorm(hidden, eps=1e-5)
        self.attn = nn.Linear(hidden, hidden)
        self.ln_2 = nn.RMSNorm(hidden)
        self.mlp = nn.Sequential(nn.Linear(hidden, 2 * hidden), nn.SiLU(),
                                 nn.Linear(2 * hidden, hidden))


def rms_stack(hidden=48, depth=3, seed=0):
    torch.manual_seed(seed)
    blocks, final = nn.ModuleList(RmsBlock(hidden) for _ in range(depth)), nn.RMSNorm(hidden)
    with torch.no_grad():
        for module in [*blocks.modules(), final]:
            if isinstance(module, nn.RMSNorm):
                module.weight.copy_(1 + 0.1 * torch.randn(hidden))
    return blocks, final


def unfused(x, blocks, final):
    for block in blocks:
        x = x + block.attn(block.ln_1(x))
        x = x + block.mlp(block.ln_2(x))
    return x, final(x)


def test_prenorm_stack_of_rms_norms():
    blocks, final = rms_stack()
    x = torch.randn(3, 5, 48)
    parameters = [*blocks.parameters(), *final.parameters()]
    results = []
    for forward in (unfused, lambda *a: prenorm_forward(*a, implementation="torch")):
        leaf = x.clone().requires_grad_()
        residual, out = forward(leaf, blocks, final)
        grads = torch.autograd.grad(residual.square().mean() + out.sin().sum(),
                                    [leaf, *parameters])
        results.append([residual, out, *grads])
    for actual, expected in zip(results[1], results[0]):
        torch.testing.assert_close(actual, expected, rtol=1e-4, atol=1e-5)


def test_prenorm_stack_with_checkpoints_runs_and_is_near():
    blocks, final = rms_stack()
    x = torch.randn(3, 5, 48)
    grads = []
    for dtype in (None, torch.int8):
        leaf = x.clone().requires_grad_()
        residual, out = prenorm_forward(leaf, blocks, final, implementation="torch",
                                        checkpoint_dtype=dtype)
        grads.append((out, *torch.autograd.grad(out.square().sum(), [leaf, final.weight])))
    assert torch.equal(grads[0][0], grads[1][0])  # the outputs are not affected
    for exact, near in zip(grads[0][1:], grads[1][1:]):
        assert not torch.equal(exact, near)
        assert (exact - near).norm() < 0.05 * exact.norm()


def test_residual_norm_takes_rms_norm_modules():
    norm = nn.RMSNorm(32)
    x, branch = torch.randn(2, 6, 32), torch.randn(2, 6, 32)
    updated, normalized = residual_norm(x, branch, norm, implementation="torch")
    assert torch.equal(updated, x + branch)
    torch.testing.assert_close(normalized, norm(x + branch))
    torch.manual_seed(3)
    updated, _ = residual_norm(x, branch, norm, 0.5, implementation="torch")
    torch.manual_seed(3)
    assert torch.equal(updated, x + F.dropout(branch, 0.5))
    assert torch.equal(residual_norm(x, branch, norm, 0.5, False, implementation="torch")[0],
                       x + branch)
    with pytest.raises(ValueError, match="hidden size 32"):
        residual_norm(x, branch, nn.RMSNorm(16), implementation="torch")
    with pytest.raises(ValueError, match="affine weight"):
        residual_norm(x, branch, nn.RMSNorm(32, elementwise_affine=False))
    with pytest.raises(ValueError, match="checkpoint_dtype needs"):
        residual_norm(x, branch, nn.LayerNorm(32), checkpoint_dtype=torch.int8)
    with pytest.raises(ValueError, match="checkpoint_dtype needs"):
        prenorm_forward(x, [object.__new__(_LayerNormBlock)], nn.LayerNorm(32),
                        checkpoint_dtype=torch.int8)


class _LayerNormBlock:
    ln_1 = nn.LayerNorm(32)


def test_no_warning_on_the_torch_path():
    x, branch, weight = make((2, 16))
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        residual_rms_norm(x, branch, weight, implementation="torch")


def check_default_eps(device, implementation, dtype, scale):
    """A module without an eps: fp32's, which PyTorch adds to the mean of a 16-bit
    stream too. Against the definition in 64 bits, and against the module: that may
    round once more (before the weight), so both are within two steps of another."""
    torch.manual_seed(4)
    norm = nn.RMSNorm(96).to(device, dtype)
    with torch.no_grad():
        norm.weight.copy_(1.0 + 0.1 * torch.randn(96))
    x, branch = ((scale * torch.randn(3, 7, 96)).to(dtype) for _ in range(2))
    with torch.no_grad():
        updated, normalized = residual_norm(x.to(device), branch.to(device), norm,
                                            implementation=implementation)
        module = norm(updated)
    assert reference.same_bits(updated, reference.update(x, branch))
    value = reference.normalized(updated.cpu(), norm.weight.detach().cpu(), 2.0 ** -23)
    reference.assert_within(normalized, value, reference.normalized_bound(value, dtype),
                            (dtype, scale))
    step = torch.finfo(dtype).eps
    torch.testing.assert_close(normalized, module, rtol=2 * step + 64 * reference.U,
                               atol=2 * reference.SUBNORMAL[dtype])


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("scale", [1.0, 0.1, 0.02, 1e-4])
def test_default_eps_is_the_modules(dtype, scale):
    check_default_eps("cpu", "torch", dtype, scale)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("scale", [1.0, 0.1, 0.02, 1e-4])
def test_default_eps_is_the_modules_on_the_gpu(dtype, scale):
    check_default_eps("cuda", "gfx950", dtype, scale)


def test_default_eps_of_an_fp64_stream():
    norm = nn.RMSNorm(32).double()
    x = 1e-8 * torch.randn(4, 32, dtype=torch.float64)
    normalized = residual_norm(x, None, norm, implementation="torch")[1]
    torch.testing.assert_close(normalized, norm(x), rtol=1e-12, atol=0)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_prenorm_stack_in_16_bits_is_the_unfused_model(dtype):
    """Modules without an eps, a small stream. The unfused model rounds at the same
    places, but for one rounding more that its 7 norms may make (half a step each);
    taken as a whole step each through sublayers of gain about one."""
    blocks, final = rms_stack()
    for module in [*blocks.modules(), final]:
        if isinstance(module, nn.RMSNorm):
            module.eps = None
        elif isinstance(module, nn.Linear):
            nn.init.zeros_(module.bias)
            module.weight.data.mul_(0.02)
    blocks, final = blocks.to(dtype), final.to(dtype)
    x = (0.02 * torch.randn(3, 5, 48)).to(dtype)
    with torch.no_grad():
        for fused, plain in zip(prenorm_forward(x, blocks, final, implementation="torch"),
                                unfused(x, blocks, final)):
            assert (fused - plain).double().norm() <= (
                7 * torch.finfo(dtype).eps * plain.double().norm())
