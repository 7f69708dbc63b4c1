"""The root-mean-square norm operators on the GPU against the 64-bit reference
(tests/rms_reference.py says what is exact and derives the bounds of the rest).

Row lengths lie on both sides of every place where the kernels change: one
vector (4 or 8 columns), one wave of them, several waves, several vectors per
lane, a short last vector, groups of 32 to 256 columns that end inside a vector.
"""

import itertools
import threading
import warnings

import pytest
import torch
import torch.utils.checkpoint
from torch import nn

import rms_reference as reference
from gfx1010_kernels import (
    _cabi,
    can_use_residual_rms_norm,
    dequantize,
    prenorm_forward,
    residual_rms_norm,
    residual_rms_norm_quantized,
)

pytestmark = pytest.mark.gpu
EPS = 1e-6
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
CODE = {F32: 0, F16: 1, BF16: 2, torch.int8: 3, torch.float8_e4m3fn: 4}
LENGTHS = [1, 2, 3, 4, 5, 6, 7, 8, 9, 10, 31, 64, 100, 127, 128, 129, 200, 254, 255, 256, 257, 384,
           510, 511, 512, 513, 514, 516, 768, 1000, 1001, 1023, 1024, 1025, 1030, 1280, 1600, 2046,
           2047, 2048, 2049, 2880, 4094, 4095, 4096, 4097, 4100, 5120, 6000, 8191, 8192, 8193,
           8194, 11008, 12289, 16383, 16384]
TYPES = list(itertools.product([F32, F16, BF16], repeat=2))


def make(shape, x_dtype, branch_dtype, weight_dtype, seed=0):
    """CPU tensors from the seed: a stream with a few far larger columns."""
    generator = torch.Generator().manual_seed(seed)
    hidden = shape[-1]
    x = torch.randn(shape, generator=generator)
    x = (x * (1.0 + 15.0 * (torch.rand(hidden, generator=generator) < 0.02))).to(x_dtype)
    branch = (0.5 * torch.randn(shape, generator=generator)).to(branch_dtype)
    weight = (1.0 + 0.1 * torch.randn(hidden, generator=generator)).to(weight_dtype)
    return x, branch, weight


def check_forward(outputs, x, branch, weight, dtype, what):
    updated, normalized = outputs
    expected = reference.update(x, branch)
    assert updated.dtype == x.dtype and normalized.dtype == dtype
    assert reference.same_bits(updated, expected), what
    value = reference.normalized(expected, weight, EPS)
    reference.assert_within(normalized, value, reference.normalized_bound(value, dtype), what)


def check_gradients(grads, u, kept, weight, upstream, branch_dtype, depth, what):
    g, gw, size, terms = reference.gradients(u, kept, weight, EPS, *upstream)
    reference.assert_within(grads[0], g, reference.gradient_bound(g, size, u.dtype),
                            f"{what}: grad_x")
    assert grads[0].dtype == u.dtype
    if branch_dtype is not None:
        assert grads[1].dtype == branch_dtype
        reference.assert_within(grads[1], g, reference.gradient_bound(g, size, branch_dtype),
                                f"{what}: grad_branch")
    if grads[-1] is not None:
        assert grads[-1].dtype == weight.dtype
        reference.assert_within(grads[-1], gw,
                                reference.weight_bound(gw, terms, depth, weight.dtype),
                                f"{what}: grad_weight")


# Forward.

@pytest.mark.parametrize("hidden", LENGTHS)
def test_forward_lengths(hidden):
    for x_dtype, rows in ((F32, 3), (BF16, 5)):
        x, branch, weight = make((rows, hidden), x_dtype, BF16, F32, hidden)
        with torch.no_grad():
            for added in (branch, None):
                outputs = residual_rms_norm(
                    x.cuda(), None if added is None else added.cuda(), weight.cuda(), EPS,
                    implementation="gfx950")
                check_forward(outputs, x, added, weight, x_dtype, (hidden, x_dtype))


@pytest.mark.parametrize("x_dtype,branch_dtype", TYPES)
@pytest.mark.parametrize("weight_dtype,dtype", TYPES)
def test_forward_types(x_dtype, branch_dtype, weight_dtype, dtype):
    for shape in ((2, 3, 136), (4, 1027), (3, 4, 2, 2048)):
        x, branch, weight = make(shape, x_dtype, branch_dtype, weight_dtype, 1)
        with torch.no_grad():
            outputs = residual_rms_norm(x.cuda(), branch.cuda(), weight.cuda(), EPS,
                                        implementation="gfx950", normalized_dtype=dtype)
        check_forward(outputs, x, branch, weight, dtype, shape)


@pytest.mark.parametrize("rows", [1, 2, 3, 4, 5, 63, 64, 65, 1023, 2049])
@pytest.mark.parametrize("hidden", [64, 513, 1024])
def test_forward_rows(rows, hidden):
    x, branch, weight = make((rows, hidden), BF16, BF16, BF16, rows)
    outputs = residual_rms_norm(x.cuda(), branch.cuda(), weight.cuda(), EPS)
    check_forward(outputs, x, branch, weight, BF16, (rows, hidden))


def variants(tensor):
    """The same values in tensors of other strides, offsets and orders."""
    rows, hidden = tensor.shape
    wide = torch.zeros(rows, 2 * hidden + 3, dtype=tensor.dtype, device="cuda")
    wide[:, 3:3 + hidden] = tensor
    yield "one part of wider rows", wide[:, 3:3 + hidden]
    for off in (1, 2):
        flat = torch.zeros(rows * hidden + off, dtype=tensor.dtype, device="cuda")
        flat[off:] = tensor.flatten()
        yield f"{off} elements off alignment", flat[off:].view(rows, hidden)
    yield "transposed", tensor.t().contiguous().t()
    spaced = torch.zeros(rows, hidden, 2, dtype=tensor.dtype, device="cuda")
    spaced[..., 1] = tensor
    yield "every second element", spaced[..., 1]
    yield "rows backwards", tensor.flip(0).contiguous().as_strided(
        (rows, hidden), (hidden, 1)).flip(0)


@pytest.mark.parametrize("hidden", [96, 514, 515, 1600])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_strides_offsets_and_orders(hidden, dtype):
    x, branch, weight = make((6, hidden), dtype, dtype, dtype, 2)
    gx, gb, gw = x.cuda(), branch.cuda(), weight.cuda()
    expected = residual_rms_norm(gx, gb, gw, EPS, implementation="gfx950")
    codes = residual_rms_norm_quantized(gx, gb, gw, EPS, group_size=64, implementation="gfx950")
    spaced = torch.zeros(hidden, 3, dtype=dtype, device="cuda")
    spaced[:, 1] = gw
    for (name, other_x), (_, other_b) in zip(variants(gx), variants(gb)):
        for w in (gw, spaced[:, 1]):
            outputs = residual_rms_norm(other_x, other_b, w, EPS, implementation="gfx950")
            for a, b in zip(outputs, expected):
                assert a.is_contiguous() and reference.same_bits(a, b), name
            for a, b in zip(residual_rms_norm_quantized(
                    other_x, other_b, w, EPS, group_size=64, implementation="gfx950"), codes):
                assert reference.same_bits(a, b), name
    # One row read by all, and a batch whose dimensions are no single run of rows.
    row = gb[:1].expand(6, hidden)
    outputs = residual_rms_norm(gx, row, gw, EPS, implementation="gfx950")
    for a, b in zip(outputs, residual_rms_norm(gx, row.contiguous(), gw, EPS)):
        assert reference.same_bits(a, b)
    batch = torch.stack([gx, gx + 1], 1)[:, :, None].expand(6, 2, 2, hidden)
    outputs = residual_rms_norm(batch, batch, gw, EPS, implementation="gfx950")
    for a, b in zip(outputs, residual_rms_norm(batch.contiguous(), batch.contiguous(), gw, EPS)):
        assert reference.same_bits(a, b)


def test_dispatch_reaches_the_kernels(recwarn):
    x, branch, weight = (t.cuda() for t in make((4, 96), BF16, BF16, BF16))
    assert can_use_residual_rms_norm(x, branch, weight)
    first = residual_rms_norm(x, branch, weight)
    again = residual_rms_norm(x, branch, weight)
    strict = residual_rms_norm(x, branch, weight, implementation="gfx1010")
    for a, b, c in zip(first, again, strict):
        assert reference.same_bits(a, b) and reference.same_bits(a, c)
    assert not [w for w in recwarn if "was not used" in str(w.message)]
    with pytest.warns(RuntimeWarning, match="hidden size must be between"):
        residual_rms_norm(torch.ones(1, 16385, device="cuda"), None,
                          torch.ones(16385, device="cuda"))
    with pytest.raises(RuntimeError, match="unsupported RMSNorm hidden size"):
        residual_rms_norm(torch.ones(1, 16385, device="cuda"), None,
                          torch.ones(16385, device="cuda"), implementation="gfx950")
    with pytest.raises(RuntimeError, match="branch must match x"):
        residual_rms_norm(x, branch[:2], weight, implementation="gfx950")
    with pytest.raises(RuntimeError, match="same HIP device|must be HIP"):
        residual_rms_norm(x, branch, weight.cpu(), implementation="gfx950")


@pytest.mark.parametrize("shape", [(0, 96), (2, 0, 96)])
def test_empty(shape):
    x = torch.zeros(shape, device="cuda", dtype=BF16, requires_grad=True)
    branch = torch.zeros(shape, device="cuda", requires_grad=True)
    weight = torch.ones(96, device="cuda", requires_grad=True)
    for checkpoint in (None, torch.int8):
        updated, normalized = residual_rms_norm(x, branch, weight, implementation="gfx950",
                                                checkpoint_dtype=checkpoint)
        assert updated.shape == normalized.shape == shape
        grads = torch.autograd.grad([updated, normalized], [x, branch, weight],
                                    [updated, normalized])
        assert grads[0].shape == shape and grads[1].dtype == F32 and not grads[2].any()
    with torch.no_grad():
        codes, scale = residual_rms_norm_quantized(x, branch, weight, group_size=64)[1:]
        assert codes.shape == shape and scale.shape == (*shape[:-1], 2)
        assert dequantize(codes, scale, group_size=64).shape == shape


# 8-bit outputs.

@pytest.mark.parametrize("hidden", LENGTHS)
@pytest.mark.parametrize("dtype", [torch.int8, torch.float8_e4m3fn])
def test_quantized_lengths(hidden, dtype):
    for x_dtype, rows, group in ((F32, 3, 64), (BF16, 5, None), (F16, 2, 128), (BF16, 4, 32),
                                 (F32, 2, None), (F32, 5, 256), (BF16, 3, 256)):
        x, branch, weight = make((rows, hidden), x_dtype, BF16, F32, hidden)
        x[-1], branch[-1] = 0, 0
        updated, codes, scale = residual_rms_norm_quantized(
            x.cuda(), branch.cuda(), weight.cuda(), EPS, dtype=dtype, group_size=group,
            implementation="gfx950")
        u = reference.update(x, branch)
        assert reference.same_bits(updated, u)
        expected, expected_scale = reference.quantized(u, weight, EPS, group, dtype)
        what = (hidden, x_dtype, group)
        assert codes.dtype == dtype and reference.same_bits(codes, expected), what
        reference.assert_within(scale, expected_scale,
                                32 * reference.U * expected_scale + 2.0 ** -149, what)
        for out in (F32, F16, BF16):
            values = dequantize(codes, scale, group_size=group, dtype=out,
                                implementation="gfx950")
            spread = reference.spread(scale.cpu(), group or hidden, hidden)
            assert reference.same_bits(values, (expected.float() * spread).to(out)), (what, out)


@pytest.mark.parametrize("x_dtype,branch_dtype", TYPES)
def test_quantized_types(x_dtype, branch_dtype):
    for weight_dtype, group in ((F32, None), (F16, 128), (BF16, 64)):
        x, branch, weight = make((2, 3, 1032), x_dtype, branch_dtype, weight_dtype, 5)
        for added in (branch, None):
            updated, codes, scale = residual_rms_norm_quantized(
                x.cuda(), None if added is None else added.cuda(), weight.cuda(), EPS,
                dtype=torch.int8, group_size=group, implementation="gfx950")
            u = reference.update(x, added)
            expected, expected_scale = reference.quantized(u, weight, EPS, group, torch.int8)
            assert reference.same_bits(updated, u) and reference.same_bits(codes, expected)
            reference.assert_within(scale, expected_scale,
                                    32 * reference.U * expected_scale, "scale")


def test_dequantize_of_other_layouts():
    codes = torch.arange(-126, 126, dtype=torch.int8).view(12, 21)
    scale = torch.rand(12, 1)
    expected = codes.float() * scale
    for a in (codes.cuda(), codes.t().contiguous().t().cuda(),
              torch.cat([codes, codes], 1).cuda()[:, :21]):
        for b in (scale.cuda(), scale.expand(12, 2).cuda()[:, :1]):
            assert torch.equal(dequantize(a, b, dtype=F32, implementation="gfx950").cpu(), expected)
    every = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).view(1, 256)
    values = dequantize(every.cuda(), torch.full((1, 1), 0.5, device="cuda"), dtype=F32)
    assert torch.equal(values.cpu().nan_to_num(7.0), (every.float() * 0.5).nan_to_num(7.0))


# Infinities, NaNs and extremes.

@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("hidden", [100, 512, 2049])
def test_rows_that_are_not_finite(bad, hidden):
    x, branch, weight = make((6, hidden), F32, F32, F32, 3)
    clean = [t.clone() for t in (x, branch)]
    x[1, 7], branch[4, hidden - 1] = bad, bad
    gx, gb, gw = x.cuda(), branch.cuda(), weight.cuda()
    good = [0, 2, 3, 5]
    before = residual_rms_norm(*(t.cuda() for t in clean), gw, EPS)
    updated, normalized = residual_rms_norm(gx, gb, gw, EPS, implementation="gfx950")
    assert torch.equal(updated.cpu().nan_to_num(9.0), (x + branch).nan_to_num(9.0))
    assert reference.same_bits(normalized[good], before[1][good])
    for row, column in ((1, 7), (4, hidden - 1)):
        assert normalized[row, column].isnan()
        others = normalized[row].cpu()[torch.arange(hidden) != column]
        assert others.isnan().all() if bad != bad else (others == 0).all()
    for dtype in (torch.int8, torch.float8_e4m3fn):
        codes, scale = residual_rms_norm_quantized(gx, gb, gw, EPS, dtype=dtype,
                                                   group_size=64, implementation="gfx950")[1:]
        values = dequantize(codes, scale, group_size=64, dtype=F32).cpu()
        assert values[good].isfinite().all()
        for row, column in ((1, 7), (4, hidden - 1)):
            group = slice(column // 64 * 64, column // 64 * 64 + 64)
            assert values[row, group].isnan().all()
            rest = torch.cat([values[row, :group.start], values[row, group.stop:]])
            assert rest.isnan().all() if bad != bad else (rest == 0).all()


@pytest.mark.parametrize("checkpoint", [None, torch.int8])
def test_gradients_of_rows_that_are_not_finite(checkpoint):
    x, branch, weight = (t.cuda() for t in make((5, 300), F32, F32, F32, 4))
    x[2, 5] = float("inf")
    upstream = [torch.randn(5, 300, device="cuda") for _ in range(2)]
    upstream[1][4, 8] = float("nan")
    leaves = [t.requires_grad_() for t in (x, branch, weight)]
    outputs = residual_rms_norm(*leaves, EPS, implementation="gfx950",
                                checkpoint_dtype=checkpoint)
    grad_x, _, grad_weight = torch.autograd.grad(outputs, leaves, upstream)
    assert grad_x[[0, 1, 3]].isfinite().all()
    assert grad_x[2].isnan().any() and grad_x[4].isnan().all()
    assert grad_weight[8].isnan()


@pytest.mark.parametrize("rows", [7, 1030])
@pytest.mark.parametrize("hidden", [20, 33, 64, 90, 128, 200, 256])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_short_rows_are_independent(rows, hidden, dtype):
    """Rows that share a wave: a row's bits are those it has among others, and a
    NaN in one stays there."""
    x, branch, weight = (t.cuda() for t in make((rows, hidden), dtype, dtype, dtype, hidden))
    upstream = [torch.randn(rows, hidden, device="cuda").to(dtype) for _ in range(2)]

    def run(order, x):
        leaves = [x[order].requires_grad_(), branch[order].requires_grad_()]
        results = []
        for checkpoint in (None, torch.int8):
            outputs = residual_rms_norm(*leaves, weight, EPS, implementation="gfx950",
                                        checkpoint_dtype=checkpoint)
            results += [*outputs, *torch.autograd.grad(outputs, leaves,
                                                       [t[order] for t in upstream])]
        for group in (None, 32, 128):
            codes, scale = residual_rms_norm_quantized(
                x[order], branch[order], weight, EPS, dtype=torch.int8, group_size=group,
                implementation="gfx950")[1:]
            results += [codes, scale, dequantize(codes, scale, group_size=group, dtype=F32)]
        return [t.detach() for t in results]

    straight = torch.arange(rows, device="cuda")
    expected = run(straight, x)
    order = torch.randperm(rows, device="cuda")
    for got, want in zip(run(order, x), expected):
        assert reference.same_bits(got, want[order])
    spoiled = x.clone()
    spoiled[2::5, hidden // 2] = float("nan")
    rest = straight[straight % 5 != 2]
    for got, want in zip(run(straight, spoiled), expected):
        assert reference.same_bits(got[rest], want[rest])


def test_extreme_magnitudes():
    """Rows whose squares overflow or vanish in fp32 go as the formula sends
    them; groups far under 2^-100 have zero codes."""
    x = torch.stack([torch.full((256,), 1e30), torch.full((256,), 1e-38), torch.zeros(256)])
    weight = torch.ones(256)
    normalized = residual_rms_norm(x.cuda(), None, weight.cuda(), EPS)[1].cpu()
    assert (normalized[0] == 0).all() and (normalized[2] == 0).all()
    torch.testing.assert_close(normalized[1], x[1] * 1e3, rtol=1e-5, atol=0)
    codes, scale = residual_rms_norm_quantized(x.cuda(), None, weight.cuda(), EPS,
                                               dtype=torch.int8)[1:]
    assert (codes[0] == 127).all() and not codes[1:].any()
    assert (scale[0] == 0).all() and scale.isfinite().all()
    half = torch.full((2, 64), 60000.0, dtype=F16)
    updated, normalized = residual_rms_norm(half.cuda(), half.cuda(), torch.ones(64).cuda(), EPS)
    assert updated.isinf().all() and normalized.isnan().all()  # as (x + branch) in fp16


# Backward.

def step(x, branch, weight, upstream, checkpoint, needs=(True, True, True), dtype=None):
    leaves = [t.cuda().requires_grad_(need) if t is not None else None
              for t, need in zip((x, branch, weight), needs)]
    outputs = residual_rms_norm(*leaves, EPS, implementation="gfx950",
                                checkpoint_dtype=checkpoint, normalized_dtype=dtype)
    wanted = [t for t in leaves if t is not None and t.requires_grad]
    given = [(o, g.cuda()) for o, g in zip(outputs, upstream) if g is not None]
    found = torch.autograd.grad([o for o, _ in given], wanted, [g for _, g in given],
                                allow_unused=True)
    grads = iter(found)
    return outputs, [next(grads) if t is not None and t.requires_grad else None for t in leaves]


def kept_of(u, checkpoint):
    return u if checkpoint is None else reference.checkpoint(u)[2]


@pytest.mark.parametrize("hidden", LENGTHS)
@pytest.mark.parametrize("checkpoint", [None, torch.int8])
def test_backward_lengths(hidden, checkpoint):
    for x_dtype, rows in ((F32, 3), (BF16, 6), (F16, 1)):
        x, branch, weight = make((rows, hidden), x_dtype, BF16, F32, hidden)
        upstream = [torch.randn(rows, hidden).to(x_dtype) for _ in range(2)]
        outputs, grads = step(x, branch, weight, upstream, checkpoint)
        check_forward(outputs, x, branch, weight, x_dtype, hidden)
        u = reference.update(x, branch)
        check_gradients(grads, u, kept_of(u, checkpoint), weight, upstream, BF16, rows,
                        (hidden, x_dtype))


@pytest.mark.parametrize("x_dtype,branch_dtype", TYPES)
@pytest.mark.parametrize("weight_dtype,dtype", TYPES)
@pytest.mark.parametrize("checkpoint", [None, torch.int8])
def test_backward_types(x_dtype, branch_dtype, weight_dtype, dtype, checkpoint):
    for shape in ((3, 2, 200), (5, 1027)):
        x, branch, weight = make(shape, x_dtype, branch_dtype, weight_dtype, 6)
        upstream = [torch.randn(shape).to(x_dtype), torch.randn(shape).to(dtype)]
        _, grads = step(x, branch, weight, upstream, checkpoint, dtype=dtype)
        u = reference.update(x, branch)
        check_gradients(grads, u, kept_of(u, checkpoint), weight, upstream, branch_dtype, 6,
                        shape)


@pytest.mark.parametrize("rows", [1, 2, 5, 127, 511, 512, 513, 1023, 1024, 1025, 4099, 20011])
@pytest.mark.parametrize("hidden,x_dtype", [(3, BF16), (65, F32), (384, F32), (1024, BF16),
                                            (2056, BF16), (4096, F16), (4097, BF16)])
def test_backward_rows(rows, hidden, x_dtype):
    if rows * hidden > 1 << 23:
        rows = (1 << 23) // hidden | 1
    x, branch, weight = make((rows, hidden), x_dtype, x_dtype, F32, rows)
    upstream = [torch.randn(rows, hidden).to(x_dtype) for _ in range(2)]
    for checkpoint in (None, torch.int8):
        _, grads = step(x, branch, weight, upstream, checkpoint)
        u = reference.update(x, branch)
        check_gradients(grads, u, kept_of(u, checkpoint), weight, upstream, x_dtype, 512,
                        (rows, hidden))
        _, again = step(x, branch, weight, upstream, checkpoint)
        assert all(reference.same_bits(a, b) for a, b in zip(grads, again))


@pytest.mark.parametrize("checkpoint", [None, torch.int8])
def test_backward_of_parts(checkpoint):
    """Each output alone, each input alone, no branch, broadcast inputs."""
    x, branch, weight = make((7, 520), BF16, F32, F32, 8)
    u = reference.update(x, branch)
    gu, gy = torch.randn(7, 520).to(BF16), torch.randn(7, 520).to(BF16)
    kept = kept_of(u, checkpoint)
    _, grads = step(x, branch, weight, (None, gy), checkpoint)
    check_gradients(grads, u, kept, weight, (None, gy), F32, 7, "normalized alone")
    _, grads = step(x, branch, weight, (gu, None), checkpoint)
    assert reference.same_bits(grads[0], gu) and torch.equal(grads[1].cpu(), gu.float())
    assert grads[2] is None
    _, all_grads = step(x, branch, weight, (gu, gy), checkpoint)
    for needs in itertools.product([True, False], repeat=3):
        if any(needs):
            _, grads = step(x, branch, weight, (gu, gy), checkpoint, needs)
            for need, grad, full in zip(needs, grads, all_grads):
                assert (reference.same_bits(grad, full) if need else grad is None), needs
    outputs, grads = step(x, None, weight, (None, gy), checkpoint)
    check_gradients([grads[0], grads[2]], x, kept_of(x, checkpoint), weight, (None, gy), None, 7,
                    "no branch")
    # x itself is an output without a branch: its gradient adds up.
    _, both = step(x, None, weight, (gu, gy), checkpoint)
    torch.testing.assert_close(both[0].float(), grads[0].float() + gu.cuda().float(), rtol=2 ** -7,
                               atol=2 ** -7)
    # A broadcast branch (its gradient is the sum over the rows) and gradients
    # of stride zero (those of sum()).
    row = branch[:1].cuda().requires_grad_()
    updated, normalized = residual_rms_norm(x.cuda(), row.expand(7, 520), weight.cuda(), EPS,
                                            checkpoint_dtype=checkpoint)
    (summed,) = torch.autograd.grad(updated.float().sum() + normalized.float().sum(), row)
    ub = reference.update(x, branch[:1].expand(7, 520))
    ones = torch.ones(7, 520)
    g, _, size, _ = reference.gradients(ub, kept_of(ub, checkpoint), weight, EPS, ones, ones)
    bound = reference.gradient_bound(g, size, F32).sum(0, keepdim=True) \
        + 7 * reference.U * g.abs().sum(0, keepdim=True)
    reference.assert_within(summed, g.sum(0, keepdim=True), bound, "broadcast branch")


def test_gradients_are_those_of_differences():
    """Along one direction of every input at once: central differences of the
    fp32 outputs' sum, taken in 64 bits. The outputs are off by at most 32 u, so
    the slope by 64 u * sum|terms| / (2 h) = 0.02 at h = 2^-6; the third
    derivative's h^2 / 6 = 4e-5 of a slope of about 30 is less."""
    x, branch, weight = (t.double() for t in make((5, 96), F32, F32, F32, 9))
    x, branch = x.clamp(-3, 3), branch.clamp(-2, 2)
    upstream = [torch.randn(5, 96), torch.randn(5, 96)]
    direction = [torch.randn(t.shape).sign().double() * 2.0 ** -2 for t in (x, branch, weight)]
    h = 2.0 ** -6

    def value(scale):
        moved = [(t + scale * d).float() for t, d in zip((x, branch, weight), direction)]
        actual = [(m.double() - t) / scale for m, t in zip(moved, (x, branch, weight))]
        outputs = residual_rms_norm(*(m.cuda() for m in moved), EPS, implementation="gfx950")
        return sum((o.cpu().double() * g.double()).sum() for o, g in zip(outputs, upstream)), actual

    plus, _ = value(h)
    minus, _ = value(-h)
    _, grads = step(x.float(), branch.float(), weight.float(), upstream, None)
    slope = sum((g.cpu().double() * d).sum() for g, d in zip(grads, direction))
    assert abs((plus - minus) / (2 * h) - slope) < 0.05 + 0.01 * abs(slope)


def test_checkpoint_is_what_it_is_documented_to_be():
    """The codes and scales bit for bit, and what the graph keeps alive."""
    from gfx1010_kernels import _C

    for hidden, x_dtype in ((1, F32), (130, F32), (1000, BF16), (16384, F16)):
        x, branch, weight = make((3, hidden), x_dtype, F32, F32, hidden)
        updated, _, state = _C.residual_rms_norm_forward(
            x.cuda(), branch.cuda(), weight.cuda(), EPS, None, True)
        codes, scale, _ = reference.checkpoint(updated.cpu())
        kept = state.cpu()
        start = 256
        found = kept[start:start + scale.numel() * 4].view(torch.float32).view(scale.shape)
        assert reference.same_bits(found, scale)
        assert torch.equal(kept[-3 * hidden:].view(torch.int8).view(3, hidden), codes)
        del updated, state
    x = torch.randn(4096, 2048, device="cuda", dtype=BF16)
    weight = torch.ones(2048, device="cuda", dtype=BF16, requires_grad=True)
    kept = {}
    for checkpoint in (None, torch.int8):
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        updated, normalized = residual_rms_norm(x, x, weight, checkpoint_dtype=checkpoint)
        del updated
        kept[checkpoint] = torch.cuda.memory_allocated() - before - normalized.nbytes
        del normalized
    assert kept[None] >= x.nbytes
    assert kept[torch.int8] <= x.nbytes // 2 * (1 + 4 / 128) + 4096 * 4 + 4096


def test_gradients_of_two_leaves_are_no_alias():
    """One tensor is handed to x and to a branch of its type; what accumulates
    in their .grad must not be shared."""
    for checkpoint in (None, torch.int8):
        x, branch, weight = (t.cuda().requires_grad_() for t in make((9, 128), BF16, BF16, BF16))
        for turn in range(2):
            updated, normalized = residual_rms_norm(x, branch, weight,
                                                    checkpoint_dtype=checkpoint)
            (updated.float().sum() + normalized.float().square().sum()).backward()
            assert reference.same_bits(x.grad, branch.grad)
            assert x.grad.data_ptr() != branch.grad.data_ptr()
        before = branch.grad.clone()
        x.grad.zero_()
        assert reference.same_bits(branch.grad, before)
    # The same tensor as both inputs: its gradient counts twice.
    (twice,) = torch.autograd.grad(residual_rms_norm(x, x, weight)[0].float().sum(), x)
    assert (twice == 2).all()


@pytest.mark.parametrize("checkpoint", [None, torch.int8])
@pytest.mark.parametrize("added", [True, False])
def test_the_graph_is_kept_and_released_as_any(checkpoint, added):
    x, branch, weight = (t.cuda().requires_grad_() for t in make((9, 200), F32, BF16, F32))
    leaves = [x, branch, weight] if added else [x, weight]

    def forward():
        return residual_rms_norm(x, branch if added else None, weight,
                                 checkpoint_dtype=checkpoint)[1].square().sum()

    loss = forward()
    first = torch.autograd.grad(loss, leaves, retain_graph=True)
    again = torch.autograd.grad(loss, leaves)
    assert all(reference.same_bits(a, b) for a, b in zip(first, again))
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(loss, leaves)
    # Saved tensors go through hooks, and a recomputed segment saves the same.
    with torch.autograd.graph.save_on_cpu():
        loss = forward()
    assert all(reference.same_bits(a, b)
               for a, b in zip(first, torch.autograd.grad(loss, leaves)))
    loss = torch.utils.checkpoint.checkpoint(forward, use_reentrant=False)
    assert all(reference.same_bits(a, b)
               for a, b in zip(first, torch.autograd.grad(loss, leaves)))


def test_two_threads_at_once():
    """Forward, backward and 8-bit calls from two host threads, each on its
    stream, equal the same calls alone."""
    cases = [tuple(t.cuda() for t in make((257, hidden), BF16, BF16, BF16, hidden))
             for hidden in (1000, 2048)]

    def work(x, branch, weight):
        leaves = [t.clone().requires_grad_() for t in (x, branch, weight)]
        outputs = residual_rms_norm(*leaves, EPS, checkpoint_dtype=torch.int8)
        grads = torch.autograd.grad(outputs, leaves, [x, branch])
        with torch.no_grad():
            codes = residual_rms_norm_quantized(x, branch, weight, EPS, group_size=64)
            return [*outputs, *grads, *codes, dequantize(*codes[1:], group_size=64)]

    expected = [work(*case) for case in cases]
    torch.cuda.synchronize()
    failures = []

    def run(case, answer):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(20):
                    found = work(*case)
            stream.synchronize()
            assert all(reference.same_bits(a, b) for a, b in zip(found, answer))
        except BaseException as error:  # reported by the main thread
            failures.append(error)

    threads = [threading.Thread(target=run, args=pair) for pair in zip(cases, expected)]
    for thread in threads:
        thread.start()
    for thread in threads:
        thread.join(timeout=60)
    assert not failures, failures


def test_transforms_and_fake_tensors_are_refused():
    """A functorch transform and a FakeTensorMode around real tensors ask for
    what the kernels cannot give; the call raises and the next one is served."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    x, branch, weight = (t.cuda() for t in make((3, 64), F32, F32, F32))
    expected = residual_rms_norm(x, branch, weight)
    with pytest.raises(Exception):
        torch.func.grad(lambda t: residual_rms_norm(t, branch, weight)[1].sum())(x)
    with pytest.raises(Exception):
        torch.func.vmap(lambda t: residual_rms_norm(t, None, weight)[1])(x)
    with FakeTensorMode(allow_non_fake_inputs=True), pytest.raises(Exception):
        residual_rms_norm(x, branch, weight)
    for a, b in zip(residual_rms_norm(x, branch, weight), expected):
        assert reference.same_bits(a, b)


def test_second_order_gradients_are_refused():
    x = torch.randn(4, 64, device="cuda", requires_grad=True)
    weight = torch.ones(64, device="cuda", requires_grad=True)
    normalized = residual_rms_norm(x, None, weight)[1]
    (grad,) = torch.autograd.grad(normalized.square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="second-order gradients"):
        grad.square().sum().backward()


def test_inplace_change_of_what_is_kept_raises():
    x = torch.randn(4, 64, device="cuda")
    weight = torch.ones(64, device="cuda", requires_grad=True)
    updated, normalized = residual_rms_norm(x, x, weight)
    updated.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        normalized.sum().backward()
    updated, normalized = residual_rms_norm(x, x, weight, checkpoint_dtype=torch.int8)
    updated.add_(1)  # nothing of it is kept
    normalized.sum().backward()


# Buffers, streams, graphs, compilation.

def guarded(count, dtype):
    """`count` elements between two runs of a pattern, and their check."""
    size = torch.empty(0, dtype=dtype).element_size()
    whole = torch.full((4096 + count * size + 4096,), 0x5A, dtype=torch.uint8, device="cuda")
    inner = whole[4096:4096 + count * size].view(dtype)

    def check():
        assert (whole[:4096] == 0x5A).all() and (whole[4096 + count * size:] == 0x5A).all()
    return inner, check


@pytest.mark.parametrize("hidden", [1, 2, 4, 6, 63, 130, 514, 516, 520, 2055, 4096, 16382, 16383])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_nothing_is_written_outside_the_outputs(hidden, dtype):
    rows, stream = 5, torch.cuda.current_stream().cuda_stream
    x, branch, weight = (t.cuda() for t in make((rows, hidden), dtype, dtype, dtype))
    count, groups = rows * hidden, -(-hidden // 128)
    buffers = dict(updated=(count, dtype), normalized=(count, dtype), rstd=(rows, F32),
                   checkpoint=(count, torch.int8), checkpoint_scale=(rows * groups, F32))
    made = {name: guarded(*spec) for name, spec in buffers.items()}
    at = {name: inner.data_ptr() for name, (inner, _) in made.items()}
    code = CODE[dtype]
    _cabi.rms_forward(x.data_ptr(), code, weight.data_ptr(), code, at["normalized"], code, rows,
                      hidden, EPS, branch=branch.data_ptr(), branch_dtype=code,
                      updated=at["updated"], rstd=at["rstd"], checkpoint=at["checkpoint"],
                      checkpoint_scale=at["checkpoint_scale"], stream=stream)
    grads = {name: guarded(*spec) for name, spec in dict(
        grad_x=(count, dtype), grad_branch=(count, F16), grad_weight=(hidden, dtype)).items()}
    workspace, check = guarded(_cabi.rms_backward_workspace_bytes(rows, hidden, code),
                               torch.uint8)
    for kept in (dict(updated=at["updated"]),
                 dict(checkpoint=at["checkpoint"], checkpoint_scale=at["checkpoint_scale"])):
        _cabi.rms_backward(x.data_ptr(), branch.data_ptr(), code, code, weight.data_ptr(), code,
                           at["rstd"], grads["grad_x"][0].data_ptr(), rows, hidden,
                           grad_branch=grads["grad_branch"][0].data_ptr(), branch_dtype=CODE[F16],
                           grad_weight=grads["grad_weight"][0].data_ptr(),
                           workspace=workspace.data_ptr(), workspace_bytes=workspace.numel(),
                           stream=stream, **kept)
    codes, code_check = guarded(count, torch.int8)
    for group in (0, 32, 128):
        scales, scale_check = guarded(rows * (1 if group == 0 else -(-hidden // group)), F32)
        values, value_check = guarded(count, dtype)
        _cabi.rms_quantize(x.data_ptr(), code, weight.data_ptr(), code, codes.data_ptr(), 3,
                           scales.data_ptr(), group, rows, hidden, EPS,
                           branch=branch.data_ptr(), branch_dtype=code, updated=at["updated"],
                           stream=stream)
        _cabi.dequantize(codes.data_ptr(), 3, scales.data_ptr(), group, values.data_ptr(), code,
                         rows, hidden, stream)
        scale_check()
        value_check()
    for inner, verify in [*made.values(), *grads.values()]:
        verify()
    check()
    code_check()


def test_another_stream_orders_the_work():
    x, branch, weight = (t.cuda() for t in make((2048, 1024), BF16, BF16, BF16))
    expected = residual_rms_norm(x, branch, weight, EPS)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        late = torch.zeros_like(x)
        for _ in range(20):
            late += 1.0  # work queued before the input is written
        late.copy_(x)
        outputs = residual_rms_norm(late, branch, weight, EPS, implementation="gfx950")
        codes = residual_rms_norm_quantized(late, branch, weight, EPS)
        values = dequantize(*codes[1:])
    side.synchronize()
    for a, b in zip(outputs, expected):
        assert reference.same_bits(a, b)
    assert (values.float() - expected[1].float()).abs().max() < 0.1 * expected[1].abs().max()


@pytest.mark.parametrize("checkpoint", [None, torch.int8])
def test_captured_steps_replay(checkpoint):
    """Two captured training steps that share the allocator's graph pool, each
    replayed several times with new inputs and eager work between."""
    x, branch, weight = (t.cuda() for t in make((130, 1000), F32, BF16, F32, 11))
    upstream = [torch.randn(130, 1000, device="cuda") for _ in range(2)]
    static = [x.clone().requires_grad_(), branch.clone().requires_grad_(),
              weight.clone().requires_grad_()]

    def work(leaves):
        outputs = residual_rms_norm(*leaves, EPS, implementation="gfx950",
                                    checkpoint_dtype=checkpoint)
        return [*outputs, *torch.autograd.grad(outputs, leaves, upstream)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work(static)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outputs = [], []
    pool = None
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=pool):
            outputs.append(work(static))
        pool = graph.pool()
        graphs.append(graph)
    for turn in range(4):
        fresh = [t.detach() + 0.25 * turn for t in (x, branch, weight)]
        with torch.no_grad():
            for leaf, value in zip(static, fresh):
                leaf.copy_(value)
        expected = work([t.clone().requires_grad_() for t in fresh])
        for graph, found in zip(graphs, outputs):
            graph.replay()
            torch.cuda.synchronize()
            assert all(reference.same_bits(a, b) for a, b in zip(found, expected)), turn


def test_captured_serving_calls_replay():
    x, branch, weight = (t.cuda() for t in make((4, 2880), BF16, BF16, BF16, 12))

    def work():
        updated, codes, scale = residual_rms_norm_quantized(x, branch, weight, EPS,
                                                            dtype=torch.int8, group_size=128)
        return [*residual_rms_norm(updated, branch, weight, EPS), codes, scale,
                dequantize(codes, scale, group_size=128)]

    work()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        found = work()
    for turn in range(3):
        x.add_(0.5)
        expected = work()
        graph.replay()
        torch.cuda.synchronize()
        assert all(reference.same_bits(a, b) for a, b in zip(found, expected)), turn


@pytest.mark.parametrize("checkpoint", [None, torch.int8])
def test_compiled_step_equals_the_eager_one(checkpoint):
    x, branch, weight = (t.cuda() for t in make((2, 9, 260), BF16, F32, F32, 13))
    upstream = [torch.randn(2, 9, 260, device="cuda").to(BF16) for _ in range(2)]

    def forward(x, branch, weight):
        first = residual_rms_norm(x, None, weight, EPS, checkpoint_dtype=checkpoint)[1]
        return residual_rms_norm(x, branch + first, weight, EPS, checkpoint_dtype=checkpoint)

    results = []
    for function in (forward, torch.compile(forward, backend="aot_eager", fullgraph=True)):
        leaves = [t.clone().requires_grad_() for t in (x, branch, weight)]
        outputs = function(*leaves)
        results.append([*outputs, *torch.autograd.grad(outputs, leaves, upstream)])
    for a, b in zip(*results):
        assert reference.same_bits(a, b)

    def serve(x, branch, weight):
        _, codes, scale = residual_rms_norm_quantized(x, branch, weight, EPS, group_size=32)
        return codes, scale, dequantize(codes, scale, group_size=32)

    with torch.no_grad():
        compiled = torch.compile(serve, backend="aot_eager", fullgraph=True)
        for a, b in zip(compiled(x, branch, weight), serve(x, branch, weight)):
            assert reference.same_bits(a, b)


def test_rows_past_two_to_the_31_elements():
    """Offsets of the last rows pass 2^31 elements (and 2^32 bytes)."""
    rows, hidden = (1 << 31) // 16384 + 3, 16384
    x = torch.zeros(rows, hidden, device="cuda", dtype=BF16)
    row, branch, weight = make((1, hidden), BF16, BF16, BF16, 14)
    x[-1] = row[0]
    added = branch.cuda().expand(rows, hidden)
    updated, normalized = residual_rms_norm(x, added, weight.cuda(), EPS, implementation="gfx950")
    check_forward((updated[-1:], normalized[-1:]), row, branch, weight, BF16, "last row")
    zero = torch.zeros(1, hidden, dtype=BF16)
    check_forward((updated[:1], normalized[:1]), zero, branch, weight, BF16, "first row")
    del normalized
    codes, scale = residual_rms_norm_quantized(x, added, weight.cuda(), EPS, dtype=torch.int8)[1:]
    expected, _ = reference.quantized(reference.update(row, branch), weight, EPS, None, torch.int8)
    assert reference.same_bits(codes[-1:], expected)
    del updated
    values = dequantize(codes, scale, dtype=BF16)
    assert torch.equal(values[-1].cpu(), (expected[0].float() * scale[-1].cpu()).to(BF16))
    del values, codes
    weight = weight.cuda().requires_grad_()
    x.requires_grad_()
    for checkpoint in (None, torch.int8):
        normalized = residual_rms_norm(x, added, weight, EPS, checkpoint_dtype=checkpoint)[1]
        upstream = torch.zeros_like(normalized)
        upstream[-1] = 1.0
        grads = torch.autograd.grad(normalized, [x, weight], upstream)
        del normalized, upstream
        u = reference.update(row, branch)
        check_gradients([grads[0][-1:], grads[1]], u, kept_of(u, checkpoint),
                        weight.detach().cpu(), (None, torch.ones(1, hidden).to(BF16)), None, 512,
                        "last row")
        assert not grads[0][:-1].any()
        del grads


def test_more_rows_than_one_grid():
    """A launch has at most 2^21 blocks; teams walk over the rows past that (of 32
    short rows or 4 longer ones per block), and so do the widening's."""
    rows, hidden = (1 << 23) + 3, 258
    row, branch, scale = make((1, hidden), BF16, BF16, BF16, 15)
    x = torch.zeros(rows, hidden, device="cuda", dtype=BF16)
    x[-1] = row[0]
    outputs = residual_rms_norm(x, branch.cuda().expand(rows, hidden), scale.cuda(), EPS,
                                implementation="gfx950")
    check_forward([t[-1:] for t in outputs], row, branch, scale, BF16, "last row")
    check_forward([t[:1] for t in outputs], torch.zeros_like(row), branch, scale, BF16, "first")
    del x, outputs
    rows, hidden = (1 << 26) + 5, 4
    generator = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(rows, hidden, device="cuda", generator=generator)
    weight = torch.randn(hidden, device="cuda", generator=generator)
    u = x + x
    normalized = residual_rms_norm(x, x, weight, EPS, implementation="gfx950")[1]
    value = reference.normalized(u, weight, EPS)
    assert ((normalized.double() - value).abs() <= 33 * reference.U * value.abs()).all()
    updated, codes, scale = residual_rms_norm_quantized(x, x, weight, EPS, dtype=torch.int8,
                                                        implementation="gfx950")
    assert torch.equal(updated, u)
    values = dequantize(codes, scale, dtype=F32)
    assert ((values - value).abs() <= 0.51 * scale).all()
    del value, values, normalized
    leaf, scale_leaf = x.clone().requires_grad_(), weight.clone().requires_grad_()
    ones = torch.ones_like(x)
    grads = torch.autograd.grad(residual_rms_norm(leaf, None, scale_leaf, EPS)[1],
                                [leaf, scale_leaf], ones)
    # 32768 places of rows/32768 = 2049 rows each, then 8 rows, 8 teams and 512 blocks.
    g, gw, size, terms = reference.gradients(x, x, weight, EPS, None, ones)
    assert ((grads[0].double() - g).abs() <= 128 * reference.U * size + reference.U * g.abs()).all()
    assert ((grads[1].double() - gw).abs() <= (32 + 2049 + 528) * reference.U * terms).all()
    del grads, g, size, ones
    rows = (1 << 29) + 1000
    codes = torch.randint(-127, 128, (rows, 1), device="cuda", dtype=torch.int8)
    scale = torch.rand(rows, 1, device="cuda")
    values = dequantize(codes, scale, dtype=F32, implementation="gfx950")
    assert torch.equal(values, codes.float().mul_(scale))


# Together, as they are used.

class Block(nn.Module):
    def __init__(self, hidden):
        super().__init__()
        self.ln_1 = nn.RMSNorm(hidden, eps=1e-5)
        self.attn = nn.Linear(hidden, hidden, bias=False)
        self.ln_2 = nn.RMSNorm(hidden, eps=1e-5)
        self.mlp = nn.Sequential(nn.Linear(hidden, 2 * hidden), nn.SiLU(),
                                 nn.Linear(2 * hidden, hidden))


@pytest.mark.parametrize("checkpoint", [None, torch.int8])
def test_training_stack(checkpoint):
    """prenorm_forward over RMSNorm blocks against the same stack through the
    PyTorch path, forward and every gradient."""
    torch.manual_seed(0)
    blocks = nn.ModuleList(Block(320) for _ in range(3)).cuda()
    final = nn.RMSNorm(320).cuda()
    x = torch.randn(4, 33, 320, device="cuda")
    parameters = [*blocks.parameters(), *final.parameters()]
    results = []
    for implementation in ("gfx950", "torch"):
        leaf = x.clone().requires_grad_()
        residual, out = prenorm_forward(leaf, blocks, final, implementation=implementation,
                                        checkpoint_dtype=checkpoint)
        loss = residual.square().mean() + out.sin().sum()
        results.append([residual, out, *torch.autograd.grad(loss, [leaf, *parameters])])
    # fp32 throughout; with the checkpoint a code next to a border may fall on
    # either side, 1/127 of one value of many.
    limit = 1e-4 if checkpoint is None else 1e-3
    for a, b in zip(*results):
        assert (a - b).norm() <= limit * b.norm()


def test_serving_stack():
    """Each norm in 8 bits, widened for a bf16 product whose output is the next
    norm's branch: against the same chain through the PyTorch path, step by step
    from the same inputs."""
    torch.manual_seed(1)
    hidden = 384
    weights = [(torch.randn(hidden, hidden, device="cuda") / hidden ** 0.5).to(BF16)
               for _ in range(4)]
    norms = [(1 + 0.1 * torch.randn(hidden, device="cuda")).to(BF16) for _ in range(4)]
    for dtype, group in ((torch.float8_e4m3fn, 128), (torch.int8, None)):
        x = torch.randn(3, 17, hidden, device="cuda").to(BF16)
        branch = None
        with torch.no_grad():
            for weight, norm in zip(weights, norms):
                options = dict(dtype=dtype, group_size=group)
                ours = residual_rms_norm_quantized(x, branch, norm, EPS, implementation="gfx950",
                                                   **options)
                plain = residual_rms_norm_quantized(x, branch, norm, EPS, implementation="torch",
                                                    **options)
                assert reference.same_bits(ours[0], plain[0])
                assert reference.same_bits(ours[1], plain[1])
                torch.testing.assert_close(ours[2], plain[2], rtol=64 * reference.U, atol=0)
                wide = dequantize(ours[1], ours[2], group_size=group, implementation="gfx950")
                exact = residual_rms_norm(x, branch, norm, EPS)[1]
                assert (wide - exact).float().norm() < 0.04 * exact.float().norm()
                x, branch = ours[0], wide @ weight


# What the calls take over from their inputs, and what they keep.

@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("added", [True, False])
@pytest.mark.parametrize("layout", ["dense", "part of wider rows", "transposed"])
def test_outputs_keep_dimension_names(layout, added, grad):
    x, branch, weight = (t.cuda() for t in make((3, 4, 96), F32, BF16, F32))
    wide = {"dense": x, "part of wider rows": torch.cat([x, x], -1)[..., :96],
            "transposed": x.transpose(0, 1).contiguous().transpose(0, 1)}[layout]
    with warnings.catch_warnings():
        warnings.simplefilter("ignore")
        named = wide.refine_names("N", "T", "C")
    leaf = named.requires_grad_(grad)
    for implementation in ("gfx950", "auto"):
        outputs = residual_rms_norm(leaf, branch if added else None, weight, EPS,
                                    implementation=implementation)
        assert [t.names for t in outputs] == [("N", "T", "C")] * 2
        plain = residual_rms_norm(x, branch if added else None, weight, EPS)
        for a, b in zip(outputs, plain):
            assert reference.same_bits(a.detach().rename(None), b)
    with torch.no_grad():
        _, codes, scale = residual_rms_norm_quantized(leaf, branch, weight, EPS, dtype=torch.int8)
        assert codes.names == ("N", "T", "C")
        assert dequantize(codes, scale, dtype=F32).names == ("N", "T", "C")


@pytest.mark.parametrize("grad,needs,expected", [(False, True, False), (True, False, False),
                                                 (True, True, True)])
def test_a_compiled_call_writes_a_checkpoint_only_where_a_gradient_is_recorded(grad, needs,
                                                                               expected):
    calls = []

    def backend(module, _):
        calls.extend(node.args[5] for node in module.graph.nodes
                     if "rms_forward" in str(node.target))
        return module.forward

    def function(x, branch, weight):
        updated, first = residual_rms_norm(x, branch, weight, EPS, checkpoint_dtype=torch.int8)
        return residual_rms_norm(updated, first, weight, EPS, checkpoint_dtype=torch.int8)

    x, branch, weight = (t.cuda() for t in make((6, 200), F32, BF16, F32))
    weight.requires_grad_(needs)
    torch._dynamo.reset()
    with torch.set_grad_enabled(grad):
        outputs = torch.compile(function, backend=backend, fullgraph=True)(x, branch, weight)
        for a, b in zip(outputs, function(x, branch, weight)):
            assert reference.same_bits(a, b) and a.requires_grad == b.requires_grad
    assert calls == [expected, expected]
    if expected:
        grads = [torch.autograd.grad(o[1].square().sum() + o[0].sin().sum(), weight)[0]
                 for o in (outputs, function(x, branch, weight))]
        assert reference.same_bits(*grads)


def test_two_threads_end():
    """As test_two_threads_at_once, of threads that are known to have ended, with
    backwards of both forms (slab blocks and the walk)."""
    cases = [tuple(t.cuda() for t in make((rows, 1000), F32, BF16, F32, rows))
             for rows in (300, 2500)]

    def work(x, branch, weight):
        leaves = [t.clone().requires_grad_() for t in (x, branch, weight)]
        outputs = residual_rms_norm(*leaves, EPS, implementation="gfx950")
        return [*outputs, *torch.autograd.grad(outputs, leaves, [x, x])]

    expected = [work(*case) for case in cases]
    torch.cuda.synchronize()
    results = {}

    def run(index):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(20):
                found = work(*cases[index])
        stream.synchronize()
        results[index] = all(reference.same_bits(a, b) for a, b in zip(found, expected[index]))

    threads = [threading.Thread(target=run, args=(index,), daemon=True) for index in range(2)]
    for thread in threads:
        thread.start()
    for thread in threads:
        thread.join(timeout=60)
        assert not thread.is_alive()
    assert results == {0: True, 1: True}


def test_what_transforms_and_fake_tensors_are_refused_for():
    """The kernels ask for addresses, which a transform's tensor does not have and
    a fake output's are null."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    x, branch, weight = (t.cuda() for t in make((3, 64), F32, F32, F32))
    residual_rms_norm(x, branch, weight)
    for implementation in ("auto", "gfx950"):
        options = dict(implementation=implementation)
        for call in (lambda t: residual_rms_norm(t, t, weight, **options)[1],
                     lambda t: residual_rms_norm(t, None, weight, **options)[1],
                     lambda t: residual_rms_norm_quantized(t, None, weight, **options)[2]):
            with pytest.raises(RuntimeError, match="data pointer"):
                torch.func.vmap(call)(x)
            with FakeTensorMode(allow_non_fake_inputs=True), pytest.raises(
                    RuntimeError, match="must not be null|data is not allocated"):
                call(x)
            assert call(x).isfinite().all()
        with pytest.raises(RuntimeError, match="data pointer"):
            torch.func.grad(lambda t: residual_rms_norm(t, branch, weight, **options)[1].sum())(x)
