"""The gated residual norm on the GPU against the 64-bit reference
(tests/gated_reference.py derives the bounds).

Row lengths lie on both sides of every place where the kernels change: one vector
(4 or 8 columns), rows that share a wave, one wave, several waves, several vectors per
lane, short last vectors.
"""

import itertools
import threading
import warnings

import pytest
import torch
import torch._dynamo.compiled_autograd as compiled_autograd
import torch.utils.checkpoint
from torch.fx.experimental.proxy_tensor import make_fx

import gated_reference as reference
from gfx1010_kernels import (
    _C,
    _cabi,
    can_use_gated_residual_rms_norm,
    gated_residual_rms_norm,
    residual_rms_norm,
)
from rms_reference import same_bits

pytestmark = pytest.mark.gpu
EPS = 1e-6
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
CODE = {F32: 0, F16: 1, BF16: 2}
LENGTHS = [1, 2, 3, 4, 7, 8, 9, 31, 64, 100, 127, 128, 129, 200, 255, 256, 257, 511, 512, 513, 514,
           768, 1001, 1024, 1025, 2047, 2048, 2880, 4095, 4096, 4097, 5120, 6001, 8191, 8192, 8193,
           8200, 11008, 12289, 16383, 16384]
NAMES = ("x", "branch", "weight", "branch_weight", "gate")
KINDS = [("none", "shared"), ("shared", "shared"), ("sample", "shared"), ("token", "shared"),
         ("none", "sample"), ("shared", "sample"), ("sample", "sample"), ("token", "sample"),
         ("token", "token")]


def to_gpu(parts):
    return [None if t is None else t.detach().cuda() for t in parts]


def call(parts, eps=EPS, **options):
    x, branch, weight, post, gate = parts
    options.setdefault("implementation", "gfx950")
    return gated_residual_rms_norm(x, branch, weight, eps, branch_weight=post, gate=gate, **options)


def step(parts, upstream, wanted=range(5), **options):
    """Outputs, and the gradients in the order of the parts (None where not wanted)."""
    parts = [None if t is None else t.detach().requires_grad_(i in wanted)
             for i, t in enumerate(parts)]
    outputs = call(parts, **options)
    places = [i for i in wanted if parts[i] is not None]
    grads = torch.autograd.grad(outputs, [parts[i] for i in places], upstream)
    found = [None] * 5
    for place, grad in zip(places, grads):
        found[place] = grad
    return outputs, found


def check(parts, upstream, what, *, backward=True, dtype=None, **options):
    given = to_gpu(parts)
    dtype = dtype or parts[0].dtype
    definition = reference.Call(parts, options.get("eps", EPS),
                                options.get("branch_eps", options.get("eps", EPS)),
                                options.get("residual_scale", 1.0),
                                options.get("branch_scale", 1.0))
    if not backward:
        with torch.no_grad():
            definition.check_forward(*call(given, normalized_dtype=dtype, **options), dtype, what)
        return
    outputs, grads = step(given, [t.cuda() for t in upstream], normalized_dtype=dtype, **options)
    definition.check_forward(*outputs, dtype, what)
    definition.check_gradients(grads, outputs[0], *upstream, what)


def upstream_of(parts, dtype, seed=0):
    generator = torch.Generator().manual_seed(seed + 100)
    return [torch.randn(parts[0].shape, generator=generator).to(kind)
            for kind in (parts[0].dtype, dtype)]


@pytest.mark.parametrize("hidden", LENGTHS)
@pytest.mark.parametrize("post", [True, False])
def test_lengths(hidden, post):
    for x_dtype, gate in ((F32, "sample"), (BF16, "none"), (F16, "token")):
        parts = reference.make((2, 3, hidden), [x_dtype, BF16, F32, x_dtype, x_dtype], post=post,
                               gate=gate, seed=hidden)
        check(parts, upstream_of(parts, x_dtype), (hidden, x_dtype))


@pytest.mark.parametrize("x_dtype,branch_dtype,dtype", itertools.product([F32, F16, BF16], repeat=3))
def test_types(x_dtype, branch_dtype, dtype):
    for index, (weight, post, gate) in enumerate(((F32, F16, BF16), (F16, BF16, F32),
                                                  (BF16, F32, F16))):
        for hidden in (72, 1027, 2048):
            parts = reference.make((2, 2, hidden), [x_dtype, branch_dtype, weight, post, gate],
                                   gate=("token", "sample", "shared")[index], seed=index)
            check(parts, upstream_of(parts, dtype), (hidden, index), dtype=dtype)


@pytest.mark.parametrize("gate,weight", KINDS)
@pytest.mark.parametrize("shape", [(1, 1, 200), (5, 1, 200), (1, 7, 200), (4, 33, 130), (3, 65, 520),
                                   (2, 300, 64), (70, 3, 96), (600, 2, 40), (130, 1, 1024)])
def test_factors(gate, weight, shape):
    for post, scales in ((True, (1.25, 0.3)), (False, (1.0, 1.0))):
        parts = reference.make(shape, [F32] * 5, post=post, gate=gate, weight=weight, seed=3)
        check(parts, upstream_of(parts, F32), (gate, weight, shape), residual_scale=scales[0],
              branch_scale=scales[1], branch_eps=1e-3)


@pytest.mark.parametrize("shape,gate,weight", [
    ((7,), "shared", "shared"), ((2, 3, 2, 24), (2, 3, 1, 24), "shared"),
    ((2, 3, 2, 24), (2, 3, 1, 24), (2, 3, 1, 24)), ((2, 3, 2, 24), (2, 1, 1, 24), "shared"),
    ((2, 3, 2, 24), (1, 24), (1, 1, 1, 24)), ((2, 1, 2, 24), (2, 1, 1, 24), (2, 1, 1, 24)),
    ((6, 24), (6, 24), (1, 24)), ((3, 1, 24), (3, 1, 24), (3, 1, 24)),
])
def test_shapes_of_factors(shape, gate, weight):
    parts = reference.make(shape, [F32] * 5, gate=gate, weight=weight, seed=4)
    check(parts, upstream_of(parts, F32), (shape, gate, weight))


@pytest.mark.parametrize("hidden", [1025, 1288, 1535, 1536, 2048, 2303, 2304, 2880, 4607, 4608, 5120,
                                    6143, 6144, 7168, 8190, 9215, 9216, 12287, 12288])
@pytest.mark.parametrize("x_dtype,branch_dtype", [(BF16, BF16), (F16, F32), (F32, F16)])
def test_launches_past_the_chip(hidden, x_dtype, branch_dtype):
    """More rows than the chip's waves take at once, where a row has fewer waves."""
    rows = 4096 // -(-hidden // 512) + 5
    for post, gate in ((True, "shared"), (hidden % 2 == 0, "token")):
        parts = reference.make((rows, hidden), [x_dtype, branch_dtype, x_dtype, F32, BF16], post=post,
                               gate=gate, seed=hidden)
        check(parts, upstream_of(parts, x_dtype), (hidden, x_dtype, gate))


@pytest.mark.parametrize("rows", [1, 2, 3, 63, 64, 65, 513, 2049])
@pytest.mark.parametrize("hidden", [24, 96, 513, 1024, 4097])
def test_rows(rows, hidden):
    parts = reference.make((rows, hidden), [BF16, BF16, BF16, BF16, BF16], gate="shared", seed=rows)
    check(parts, upstream_of(parts, BF16), (rows, hidden))


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
    yield "rows backwards", tensor.flip(0).contiguous().flip(0)
    spaced = torch.zeros(rows, hidden, 2, dtype=tensor.dtype, device="cuda")
    spaced[..., 1] = tensor
    yield "every second element", spaced[..., 1]


@pytest.mark.parametrize("hidden", [90, 514, 515, 1600])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_strides_offsets_and_orders(hidden, dtype):
    parts = to_gpu(reference.make((6, hidden), [dtype] * 5, gate="token", seed=2))
    upstream = [t.cuda() for t in upstream_of(parts, dtype)]
    expected = step(parts, upstream)
    spread = torch.zeros(hidden, 3, dtype=dtype, device="cuda")
    for versions in zip(*(variants(t) for t in (parts[0], parts[1], parts[4]))):
        (name, x), (_, branch), (_, gate) = versions
        for index in (2, 3):
            spread[:, index - 1] = parts[index]
        found = step([x, branch, spread[:, 1], spread[:, 2], gate], upstream)
        for a, b in zip([*found[0], *found[1]], [*expected[0], *expected[1]]):
            assert a.is_contiguous() and same_bits(a, b), name
        other = [dict(variants(t))[name] for t in upstream]
        for a, b in zip(step([x, branch, *parts[2:]], other)[1], expected[1]):
            assert same_bits(a, b), name


def test_broadcast_inputs_get_the_sums_of_their_gradients():
    """x, branch and gate that are expanded: strides of zero."""
    x, branch, weight, post, _ = reference.make((1, 1, 60), [F32] * 5, gate="none", seed=5)
    gate = torch.randn(4, 1, 60)
    whole = [x.expand(4, 5, 60).contiguous(), branch.expand(4, 5, 60).contiguous(), weight, post,
             gate.expand(4, 5, 60).contiguous()]
    upstream = upstream_of(whole, F32)
    definition = reference.Call(whole, EPS, EPS, 1.0, 1.0)
    leaves = [t.cuda().requires_grad_() for t in (x, branch, gate)]
    outputs = call([leaves[0].expand(4, 5, 60), leaves[1].expand(4, 5, 60), weight.cuda(),
                    post.cuda(), leaves[2].expand(4, 5, 60)])
    grads = torch.autograd.grad(outputs, leaves, [t.cuda() for t in upstream])
    expected = definition.gradients(outputs[0], *upstream)
    for grad, leaf, (value, off) in zip(grads, (x, branch, gate), (expected[0], expected[1],
                                                                   expected[4])):
        total, bound = value.sum_to_size(leaf.shape), off.sum_to_size(leaf.shape)
        sizes = value.abs().sum_to_size(leaf.shape)
        # torch's own sum over the repeats: 20 additions at most, and each term's rounding
        assert ((grad.cpu().double() - total).abs() <= bound + 22 * 2.0 ** -24 * sizes).all()


def test_dispatch_reaches_the_kernels(recwarn):
    parts = to_gpu(reference.make((2, 3, 64), [BF16] * 5))
    expected = call(parts)
    assert can_use_gated_residual_rms_norm(*parts[:3], branch_weight=parts[3], gate=parts[4])
    for implementation in ("auto", "gfx1010"):
        for a, b in zip(call(parts, implementation=implementation), expected):
            assert same_bits(a, b)
    assert not recwarn.list
    gate = torch.randn(3, 64, device="cuda")  # repeats over the first dimension
    with pytest.warns(RuntimeWarning, match="must repeat over the last"):
        gated_residual_rms_norm(*parts[:3], gate=gate)
    assert not can_use_gated_residual_rms_norm(*parts[:3], gate=gate)
    with pytest.raises(RuntimeError, match="must repeat over the last"):
        gated_residual_rms_norm(*parts[:3], gate=gate, implementation="gfx950")
    wide = torch.zeros(2, 16385, device="cuda")
    with pytest.warns(RuntimeWarning, match="hidden size"):
        gated_residual_rms_norm(wide, wide, wide[0])
    with pytest.raises(RuntimeError, match="hidden size"):
        gated_residual_rms_norm(wide, wide, wide[0], implementation="gfx950")
    with pytest.raises(RuntimeError, match="must be HIP tensors"):
        gated_residual_rms_norm(parts[0], parts[1], parts[2].cpu(), implementation="gfx950")
    with pytest.raises(RuntimeError, match="eps"):
        call(parts, eps=-1.0)
    with pytest.raises(RuntimeError, match="finite"):
        call(parts, branch_scale=float("nan"))


@pytest.mark.parametrize("shape", [(0, 64), (2, 0, 64), (0, 5, 64)])
def test_empty(shape):
    gate = torch.randn(*shape[:1], *[1] * (len(shape) - 2), 64, device="cuda", requires_grad=True)
    x = torch.zeros(shape, device="cuda", requires_grad=True)
    weight = torch.ones(64, device="cuda", requires_grad=True)
    post = torch.ones(64, device="cuda", requires_grad=True)
    outputs = call([x, x, weight, post, gate])
    assert all(t.shape == x.shape for t in outputs)
    grads = torch.autograd.grad(sum(t.sum() for t in outputs), [x, weight, post, gate])
    for grad, leaf in zip(grads, (x, weight, post, gate)):
        assert grad.shape == leaf.shape and not grad.any()


@pytest.mark.parametrize("wanted", [w for n in (1, 2) for w in itertools.combinations(range(5), n)])
def test_parts_of_the_gradient(wanted):
    parts = to_gpu(reference.make((3, 4, 136), [F32, BF16, F32, F32, F32], seed=6))
    upstream = [t.cuda() for t in upstream_of(parts, F32)]
    expected = step(parts, upstream)[1]
    for found, want in zip(step(parts, upstream, wanted)[1], expected):
        assert found is None or same_bits(found, want)


@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("gate", ["sample", "token"])
def test_one_output_alone(which, gate):
    """Without the other's gradient; the last norm's weight has none without it."""
    parts = reference.make((3, 4, 136), [F32] * 5, gate=gate, seed=7)
    upstream = upstream_of(parts, F32)
    leaves = [t.cuda().requires_grad_() for t in parts]
    outputs = call(leaves)
    grads = torch.autograd.grad(outputs[which], leaves, upstream[which].cuda(), allow_unused=True)
    assert (grads[2] is None) == (which == 0)
    given = [upstream[0], None] if which == 0 else [None, upstream[1]]
    reference.Call(parts, EPS, EPS, 1.0, 1.0).check_gradients(grads, outputs[0], *given, which)


def test_gradients_are_those_of_differences():
    """Central differences of the forward itself, in fp32: the outputs' rounding,
    32 u of values near 1 summed over 96 products, over steps of 2^-6, against third
    derivatives of the order of 10 times the step squared."""
    parts = to_gpu(reference.make((2, 2, 24), [F32] * 5, seed=8))
    parts[0].clamp_(-2, 2)
    generator = torch.Generator().manual_seed(9)
    upstream = [torch.randn(2, 2, 24, generator=generator).cuda() for _ in range(2)]
    _, grads = step(parts, upstream)
    h = 2.0 ** -6
    for index in range(5):
        direction = torch.randn(parts[index].shape, generator=generator).cuda()
        direction /= direction.norm()

        def value(sign):
            moved = list(parts)
            moved[index] = parts[index] + sign * h * direction
            return sum((o.double() * g.double()).sum() for o, g in zip(call(moved), upstream))

        slope = (value(1) - value(-1)) / (2 * h)
        along = (grads[index].double() * direction.double()).sum()
        scale = sum(g.double().norm() for g in upstream)
        assert abs(slope - along) <= 20 * h * h * scale, NAMES[index]


# Infinities, NaNs, extremes.

@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
@pytest.mark.parametrize("hidden", [60, 512, 2049])
@pytest.mark.parametrize("gate", ["sample", "token"])
def test_rows_that_are_not_finite_stay_alone(bad, hidden, gate):
    parts = to_gpu(reference.make((2, 5, hidden), [F32] * 5, gate=gate, seed=10))
    upstream = [t.cuda() for t in upstream_of(parts, F32)]
    clean = step(parts, upstream)
    spoiled = [t.clone() for t in parts]
    spoiled[0][0, 1, 7] = bad
    spoiled[1][1, 3, hidden - 1] = bad
    found = step(spoiled, upstream)
    keep = torch.ones(2, 5, dtype=torch.bool, device="cuda")
    keep[0, 1] = keep[1, 3] = False
    for a, b in zip([*found[0], *found[1][:2]], [*clean[0], *clean[1][:2]]):
        assert same_bits(a[keep], b[keep])
    assert not found[0][1][0, 1, 7].isfinite() or bad != bad
    assert found[0][1][0, 1, 7].isnan() and found[0][0][1, 3].isnan().any()
    assert not found[1][2].isfinite().all()


@pytest.mark.parametrize("rows", [1, 3, 5])
def test_infinite_factors_reach_only_their_rows(rows):
    """Teams and lanes without a row multiply no factor into a sum."""
    for hidden in (24, 130, 1030):
        parts = to_gpu(reference.make((2, rows, hidden), [F32] * 5, gate="sample", weight="sample",
                                      seed=11))
        upstream = [t.cuda() for t in upstream_of(parts, F32)]
        clean = step(parts, upstream)
        parts[2][1, 0, 3] = float("inf")
        parts[4][1, 0, 2] = float("inf")
        found = step(parts, upstream)
        for a, b in zip([*found[0], found[1][0], found[1][1], found[1][2], found[1][4]],
                        [*clean[0], clean[1][0], clean[1][1], clean[1][2], clean[1][4]]):
            assert same_bits(a[0], b[0])


def test_extreme_magnitudes():
    """Branches whose squares vanish go as the formula sends them; a zero branch
    with an eps adds nothing."""
    parts = to_gpu(reference.make((4, 96), [F32] * 5, gate="none", seed=12))
    parts[1][0] = 0.0
    parts[1][1] *= 1e-30
    parts[1][2] *= 1e15
    outputs = call(parts)
    assert same_bits(outputs[0][0], parts[0][0])
    definition = reference.Call([None if t is None else t.cpu() for t in parts], EPS, EPS, 1.0, 1.0)
    definition.check_forward(*outputs, F32, "extremes")
    assert call(parts, branch_eps=0.0)[0][0].isnan().all()  # 0 / 0


@pytest.mark.parametrize("rows", [7, 1030])
@pytest.mark.parametrize("hidden", [20, 33, 64, 128, 200, 256])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_short_rows_are_independent(rows, hidden, dtype):
    parts = to_gpu(reference.make((rows, hidden), [dtype] * 5, gate="token", seed=hidden))
    upstream = [t.cuda() for t in upstream_of(parts, dtype)]
    order = torch.randperm(rows, device="cuda")

    def run(at):
        given = [parts[0][at], parts[1][at], parts[2], parts[3], parts[4][at]]
        outputs, grads = step(given, [t[at] for t in upstream])
        return [*outputs, grads[0], grads[1], grads[4]]

    for a, b in zip(run(order), run(torch.arange(rows, device="cuda"))):
        assert same_bits(a, b[order])


# The graph, threads, streams, buffers.

def test_sums_are_the_same_on_every_run():
    parts = to_gpu(reference.make((6, 700, 768), [F32, BF16, F32, F32, F32], seed=13))
    upstream = [t.cuda() for t in upstream_of(parts, F32)]
    first = step(parts, upstream)[1]
    for _ in range(3):
        assert all(same_bits(a, b) for a, b in zip(step(parts, upstream)[1], first))


def test_the_graph_is_kept_and_released_as_any():
    leaves = [t.requires_grad_() for t in to_gpu(reference.make((3, 4, 200), [F32] * 5, seed=14))]

    def forward():
        return call(leaves)[1].square().sum()

    loss = forward()
    first = torch.autograd.grad(loss, leaves, retain_graph=True)
    again = torch.autograd.grad(loss, leaves)
    assert all(same_bits(a, b) for a, b in zip(first, again))
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(loss, leaves)
    with torch.autograd.graph.save_on_cpu():
        loss = forward()
    assert all(same_bits(a, b) for a, b in zip(first, torch.autograd.grad(loss, leaves)))
    loss = torch.utils.checkpoint.checkpoint(forward, use_reentrant=False)
    assert all(same_bits(a, b) for a, b in zip(first, torch.autograd.grad(loss, leaves)))


def test_second_order_gradients_are_refused():
    leaves = [t.requires_grad_() for t in to_gpu(reference.make((3, 4, 64), [F32] * 5))]
    grads = torch.autograd.grad(call(leaves)[1].square().sum(), leaves, create_graph=True)
    with pytest.raises(RuntimeError, match="second-order gradients"):
        grads[4].square().sum().backward()


def test_inplace_change_of_what_is_kept_raises():
    for index in (0, 1):
        parts = to_gpu(reference.make((3, 4, 64), [F32] * 5))
        parts[2].requires_grad_()
        outputs = call(parts)
        (outputs[0] if index == 0 else parts[1]).add_(1)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            outputs[1].sum().backward()


def test_the_same_tensor_as_several_inputs():
    x = torch.randn(3, 64, device="cuda", requires_grad=True)
    w = torch.rand(64, device="cuda", requires_grad=True)
    outputs = call([x, x, w, w, x])
    grads = torch.autograd.grad(outputs, [x, w], [torch.ones_like(x)] * 2)
    leaves = [x, x, w, w, x]
    leaves = [t.detach().clone().requires_grad_() for t in leaves]
    parts = torch.autograd.grad(call(leaves), leaves, [torch.ones_like(x)] * 2)
    assert same_bits(grads[1], parts[2] + parts[3])
    assert torch.allclose(grads[0], parts[0] + parts[1] + parts[4], rtol=1e-5, atol=1e-5)


def test_forward_mode_takes_the_torch_path():
    parts = to_gpu(reference.make((3, 4, 64), [F32] * 5))
    with torch.autograd.forward_ad.dual_level():
        parts[4] = torch.autograd.forward_ad.make_dual(parts[4], torch.ones_like(parts[4]))
        with pytest.warns(RuntimeWarning, match="forward-mode"):
            outputs = call(parts, implementation="auto")
        assert torch.autograd.forward_ad.unpack_dual(outputs[1]).tangent is not None
        with pytest.raises(RuntimeError, match="forward-mode"):
            call(parts)


def test_outputs_keep_dimension_names():
    parts = to_gpu(reference.make((3, 4, 64), [F32] * 5, gate="none"))
    expected = call(parts)
    with warnings.catch_warnings():
        warnings.simplefilter("ignore")
        named = parts[0].refine_names("batch", "token", "channel")
        for a, b in zip(call([named, *parts[1:]]), expected):
            assert a.names == named.names and same_bits(a.rename(None), b)


def test_two_threads_at_once():
    cases = [to_gpu(reference.make((3, 129, hidden), [BF16] * 5, seed=hidden))
             for hidden in (1000, 2048)]

    def work(parts):
        outputs, grads = step(parts, [parts[0], parts[1]])
        return [*outputs, *grads]

    expected = [work(case) for case in cases]
    torch.cuda.synchronize()
    failures = []

    def run(case, answer):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(20):
                    found = work(case)
            stream.synchronize()
            assert all(same_bits(a, b) for a, b in zip(found, answer))
        except BaseException as error:  # reported by the main thread
            failures.append(error)

    threads = [threading.Thread(target=run, args=pair) for pair in zip(cases, expected)]
    for thread in threads:
        thread.start()
    for thread in threads:
        thread.join(timeout=60)
        assert not thread.is_alive()
    assert not failures, failures


def test_another_stream_orders_the_work():
    parts = to_gpu(reference.make((4, 512, 1024), [BF16] * 5, seed=15))
    upstream = [t.cuda() for t in upstream_of(parts, BF16)]
    expected = step(parts, upstream)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        late = torch.zeros_like(parts[0])
        for _ in range(20):
            late += 1.0  # work queued before the input is written
        late.copy_(parts[0])
        found = step([late, *parts[1:]], upstream)
    side.synchronize()
    for a, b in zip([*found[0], *found[1]], [*expected[0], *expected[1]]):
        assert same_bits(a, b)


def guarded(count, dtype):
    """`count` elements between two runs of a pattern, and their check."""
    size = torch.empty(0, dtype=dtype).element_size()
    whole = torch.full((4096 + count * size + 4096,), 0x5A, dtype=torch.uint8, device="cuda")
    inner = whole[4096:4096 + count * size].view(dtype)

    def verify():
        assert (whole[:4096] == 0x5A).all() and (whole[4096 + count * size:] == 0x5A).all()
    return inner, verify


@pytest.mark.parametrize("hidden", [1, 2, 6, 63, 130, 255, 514, 516, 2055, 4096, 8194, 16383])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("gate_rows,weight_rows", [(1, 6), (3, 3), (6, 3), (6, 6), (1, 1)])
def test_nothing_is_written_outside_the_outputs(hidden, dtype, gate_rows, weight_rows):
    rows, code = 6, CODE[dtype]
    stream = torch.cuda.current_stream().cuda_stream
    generator = torch.Generator(device="cuda").manual_seed(hidden)

    def random(*shape):
        return torch.randn(*shape, device="cuda", generator=generator).to(dtype)

    x, branch, post = random(rows, hidden), random(rows, hidden), random(hidden)
    gate, weight = random(rows // gate_rows, hidden), random(rows // weight_rows, hidden)
    factors = [_cabi.RlnFactor(t.data_ptr(), code, hidden, each)
               for t, each in ((gate, gate_rows), (weight, weight_rows))]
    count = rows * hidden
    library = _cabi.library()
    outputs = [guarded(count, dtype), guarded(count, dtype), guarded(2 * rows, F32)]
    at = [inner.data_ptr() for inner, _ in outputs]
    assert library.rln_gated_forward(
        x.data_ptr(), code, hidden, branch.data_ptr(), code, hidden, post.data_ptr(), code,
        *factors, at[0], at[1], code, at[2], rows, hidden, 1.0, 1.0, EPS, EPS, stream) == 0
    grads = [guarded(size, dtype) for size in (count, count, gate.numel(), hidden, weight.numel())]
    bytes_ = library.rln_gated_backward_workspace_bytes(rows, hidden, code, gate_rows, weight_rows)
    workspace, verify = guarded(bytes_, torch.uint8)
    assert library.rln_gated_backward(
        x.data_ptr(), branch.data_ptr(), code, at[0], code, branch.data_ptr(), code, hidden,
        post.data_ptr(), code, *factors, at[2], *(inner.data_ptr() for inner, _ in grads), rows,
        hidden, 1.0, 1.0, workspace.data_ptr(), bytes_, stream) == 0
    torch.cuda.synchronize()
    for _, check_ in [*outputs, *grads, (None, verify)]:
        check_()
    # Everything inside was written: the same as through the module.
    shape = (rows // gate_rows, gate_rows, hidden) if gate_rows < rows else (
        rows // weight_rows, weight_rows, hidden)

    def repeated(t, each):
        if each == rows:
            return t[0]
        return t if each == 1 else t.view(rows // each, 1, hidden)

    if 1 in (gate_rows, weight_rows):
        shape = (rows, hidden)
    parts = [x.view(shape), branch.view(shape), repeated(weight, weight_rows), post,
             repeated(gate, gate_rows)]
    found = step(parts, [x.view(shape), branch.view(shape)])
    for (inner, _), want in zip([outputs[0], outputs[1], *grads],
                                [*found[0], found[1][0], found[1][1], found[1][4], found[1][3],
                                 found[1][2]]):
        assert same_bits(inner, want.flatten())


# Graphs, compilation, traces.

def test_captured_steps_replay():
    """Two captured training steps that share the allocator's graph pool, each
    replayed several times with new inputs and eager work between."""
    parts = to_gpu(reference.make((5, 26, 1000), [F32, BF16, F32, F32, F32], seed=16))
    upstream = [t.cuda() for t in upstream_of(parts, F32)]
    static = [t.clone().requires_grad_() for t in parts]

    def work(leaves):
        outputs = call(leaves, implementation="auto")
        return [*outputs, *torch.autograd.grad(outputs, leaves, upstream)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work(static)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outputs, pool = [], [], None
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=pool):
            outputs.append(work(static))
        pool = graph.pool()
        graphs.append(graph)
    for turn in range(4):
        fresh = [t.detach() + 0.25 * turn for t in parts]
        with torch.no_grad():
            for leaf, value in zip(static, fresh):
                leaf.copy_(value)
        expected = work([t.clone().requires_grad_() for t in fresh])
        for graph, found in zip(graphs, outputs):
            graph.replay()
            torch.cuda.synchronize()
            assert all(same_bits(a, b) for a, b in zip(found, expected)), turn


@pytest.mark.parametrize("hidden", [8200, 16384])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_captured_steps_of_long_rows(hidden, dtype):
    """Rows whose sums are in LDS, more of it than a launch has by default."""
    parts = to_gpu(reference.make((3, 5, hidden), [dtype] * 5, seed=23))
    upstream = [t.cuda() for t in upstream_of(parts, dtype)]
    static = [t.clone().requires_grad_() for t in parts]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outputs = call(static, implementation="auto")
        found = [*outputs, *torch.autograd.grad(outputs, static, upstream)]
    for turn in range(3):
        with torch.no_grad():
            for leaf, value in zip(static, parts):
                leaf.copy_(value + 0.25 * turn)
        leaves = [(t + 0.25 * turn).requires_grad_() for t in parts]
        outputs = call(leaves)
        expected = [*outputs, *torch.autograd.grad(outputs, leaves, upstream)]
        graph.replay()
        torch.cuda.synchronize()
        assert all(same_bits(a, b) for a, b in zip(found, expected)), turn


@pytest.mark.parametrize("post,gate", [(True, "sample"), (False, "token"), (True, "none")])
def test_compiled_step_equals_the_eager_one(post, gate):
    parts = to_gpu(reference.make((2, 9, 260), [BF16, F32, F32, F32, F32], post=post, gate=gate,
                                  seed=17))
    upstream = [t.cuda() for t in upstream_of(parts, BF16)]

    def forward(*given):
        it = iter(given)
        return call([None if t is None else next(it) for t in parts], implementation="auto",
                    branch_scale=0.5)

    results = []
    for function in (forward, torch.compile(forward, backend="aot_eager", fullgraph=True)):
        leaves = [t.clone().requires_grad_() for t in parts if t is not None]
        outputs = function(*leaves)
        results.append([*outputs, *torch.autograd.grad(outputs, leaves, upstream)])
    for a, b in zip(*results):
        assert same_bits(a, b)
    # Only some gradients, and only one output's.
    leaves = [t.clone().requires_grad_(i == 1) for i, t in enumerate(parts) if t is not None]
    for output in (0, 1):
        grads = [torch.autograd.grad(f(*leaves)[output], leaves[1], upstream[output])[0]
                 for f in (forward, torch.compile(forward, backend="aot_eager", fullgraph=True))]
        assert same_bits(*grads)


@pytest.mark.parametrize("implementation", ["auto", "gfx950", "torch"])
def test_traces_hold_the_operator(implementation):
    parts = to_gpu(reference.make((2, 4, 96), [F32] * 5, seed=18))
    call(parts)

    def function(*given):
        return call(given, implementation=implementation)

    expected = function(*parts)
    fresh = [t + 0.5 for t in parts]
    with torch.no_grad(), warnings.catch_warnings():
        warnings.simplefilter("ignore")
        for graph in (torch.jit.trace(function, parts), make_fx(function)(*parts)):
            for given, want in ((parts, expected), (fresh, function(*fresh))):
                for a, b in zip(graph(*given), want):
                    assert same_bits(a, b) if implementation != "torch" else torch.allclose(a, b)
    with pytest.raises(RuntimeError, match="recorded into a graph"):
        make_fx(lambda *given: _C.gated_residual_rms_norm(*given, EPS, EPS, 1.0, 1.0, None))(*parts)


@pytest.mark.parametrize("post,gate", [(True, "sample"), (False, "none"), (True, "token")])
def test_compiled_autograd(post, gate):
    def grads(seed, backend):
        torch._dynamo.reset()
        parts = to_gpu(reference.make((2, 6, 200), [F32, BF16, F32, F32, F32], post=post, gate=gate,
                                      seed=seed))
        leaves = [None if t is None else t.requires_grad_() for t in parts]
        updated, normalized = call(leaves, implementation="auto")
        loss = updated.sin().sum() + normalized.square().sum()
        if backend is None:
            loss.backward()
        else:
            with compiled_autograd._enable(torch.compile(backend=backend)):
                loss.backward()
        return [t.grad for t in leaves if t is not None]

    for seed in (0, 1):
        for backend in ("eager", "aot_eager"):
            for a, b in zip(grads(seed, backend), grads(seed, None)):
                assert same_bits(a, b)


def test_transforms_and_fake_tensors_are_refused():
    from torch._subclasses.fake_tensor import FakeTensorMode

    parts = to_gpu(reference.make((2, 3, 64), [F32] * 5))
    expected = call(parts)
    with pytest.raises(Exception):
        torch.func.grad(lambda t: call([t, *parts[1:]])[1].sum())(parts[0])
    with pytest.raises(Exception):
        torch.func.vmap(lambda t: call([t, t, *parts[2:4], None])[1])(parts[0])
    with FakeTensorMode(allow_non_fake_inputs=True), pytest.raises(Exception):
        call(parts)
    for a, b in zip(call(parts), expected):
        assert same_bits(a, b)


# Large calls.

def test_rows_past_two_to_the_31_elements():
    """Offsets of the last rows pass 2^31 elements (and 2^32 bytes)."""
    rows, hidden = (1 << 31) // 16384 + 3, 16384
    one = reference.make((1, hidden), [BF16] * 5, gate="shared", seed=19)
    x = torch.zeros(rows, hidden, device="cuda", dtype=BF16)
    x[-1] = one[0][0]
    branch = one[1].cuda().expand(rows, hidden)
    weight, post, gate = (t.cuda().requires_grad_() for t in one[2:])
    x.requires_grad_()
    outputs = call([x, branch, weight, post, gate])
    definition = reference.Call(one, EPS, EPS, 1.0, 1.0)
    definition.check_forward(*(t[-1:] for t in outputs), BF16, "last row")
    zero = reference.Call([torch.zeros_like(one[0]), *one[1:]], EPS, EPS, 1.0, 1.0)
    zero.check_forward(*(t[:1] for t in outputs), BF16, "first row")
    upstream = torch.zeros(rows, hidden, device="cuda", dtype=BF16)
    upstream[-1] = 1.0
    last = outputs[0][-1:].detach()
    grads = torch.autograd.grad(outputs[1], [x, weight, post, gate], upstream)
    assert not grads[0][:-1].any()
    definition.check_gradients([grads[0][-1:], None, *grads[1:]], last, None,
                               torch.ones(1, hidden, dtype=BF16), "last row")


def test_more_rows_than_one_grid():
    """A launch has at most 2^21 blocks; teams walk over the rows past that, and a
    backward with a sum for every pair of rows over its units."""
    rows, hidden = (1 << 23) + 3, 258
    one = reference.make((1, hidden), [BF16] * 5, gate="none", seed=20)
    x = torch.zeros(rows, hidden, device="cuda", dtype=BF16)
    x[-1] = one[0][0]
    outputs = call([x, one[1].cuda().expand(rows, hidden), one[2].cuda(), one[3].cuda(), None])
    reference.Call(one, EPS, EPS, 1.0, 1.0).check_forward(*(t[-1:] for t in outputs), BF16, "last")
    del x, outputs
    samples, hidden = (1 << 21) + 2, 8
    generator = torch.Generator(device="cuda").manual_seed(21)
    x = torch.randn(samples, 2, hidden, device="cuda", generator=generator).requires_grad_()
    gate = torch.randn(samples, 1, hidden, device="cuda", generator=generator).requires_grad_()
    weight = torch.rand(hidden, device="cuda", generator=generator)
    outputs = call([x, x.detach(), weight, None, gate])
    upstream = torch.randn(samples, 2, hidden, device="cuda", generator=generator)
    found = torch.autograd.grad(outputs[0], [x, gate], upstream)
    assert same_bits(found[0], upstream)
    expected = (upstream.double() * x.detach().double()).sum(1, keepdim=True)
    sizes = (upstream * x.detach()).abs().sum(1, keepdim=True)
    assert ((found[1].double() - expected).abs() <= 6 * 2.0 ** -24 * sizes).all()


def test_without_gate_and_weight_it_is_the_residual_norm():
    """The same sum, rounding and norm as residual_rms_norm's, bit for bit."""
    for dtype in (F32, BF16):
        x, branch, weight, _, _ = to_gpu(reference.make((33, 1000), [dtype] * 5, seed=22))
        for a, b in zip(call([x, branch, weight, None, None]),
                        residual_rms_norm(x, branch, weight, EPS, implementation="gfx950")):
            assert same_bits(a, b)


@pytest.mark.parametrize("dynamic", [None, True])
def test_compiled_calls_of_several_scales(dynamic):
    """A number that changes from call to call becomes a symbol of the compiled graph."""
    parts = to_gpu(reference.make((2, 3, 64), [F32] * 5, seed=31))
    upstream = [torch.randn_like(parts[0]) for _ in range(2)]

    def function(*given, residual_scale, branch_scale, eps):
        x, branch, weight, post, gate = given
        return gated_residual_rms_norm(
            x, branch, weight, eps, branch_weight=post, gate=gate, branch_eps=2 * eps,
            residual_scale=residual_scale, branch_scale=branch_scale)

    torch._dynamo.reset()
    compiled = torch.compile(function, backend="aot_eager", fullgraph=True, dynamic=dynamic)
    for number in (1.0, 0.5, 0.22, 3.0):
        options = dict(residual_scale=number, branch_scale=1.0 - number / 4, eps=number * 1e-6)
        found = []
        for run in (function, compiled):
            leaves = [t.clone().requires_grad_() for t in parts]
            outputs = run(*leaves, **options)
            found.append([*outputs, *torch.autograd.grad(outputs, leaves, upstream)])
        for a, b in zip(*found):
            assert same_bits(a, b), number


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("which", ["residual_scale", "branch_scale"])
def test_scales_that_are_not_finite_take_the_torch_path(bad, which):
    parts = to_gpu(reference.make((2, 3, 64), [F32] * 5, seed=31))
    with pytest.warns(RuntimeWarning, match="must be finite"):
        gated_residual_rms_norm(*parts[:3], **{which: bad})
    with pytest.raises(RuntimeError, match="must be finite"):
        gated_residual_rms_norm(*parts[:3], **{which: bad}, implementation="gfx950")


def test_what_transforms_and_fake_tensors_are_refused_for():
    """The kernels ask for addresses, which a transform's tensor does not have and a fake output's
    are null."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    parts = to_gpu(reference.make((2, 3, 64), [F32] * 5, gate="shared"))
    call(parts, implementation="auto")
    for implementation in ("auto", "gfx950"):
        options = dict(implementation=implementation)
        for place in range(5):
            with pytest.raises(RuntimeError, match="data pointer"):
                torch.func.grad(lambda t: call([*parts[:place], t, *parts[place + 1:]],
                                               **options)[1].sum())(parts[place])
        with pytest.raises(RuntimeError, match="data pointer"):
            torch.func.vmap(lambda t, b: call([t, b, *parts[2:]], **options)[1])(*parts[:2])
        with FakeTensorMode(allow_non_fake_inputs=True), pytest.raises(
                RuntimeError, match="must not be null|data is not allocated"):
            call(parts, **options)
        assert call(parts, **options)[1].isfinite().all()


@pytest.mark.parametrize("gate", ["none", "shared", "token"])
@pytest.mark.parametrize("shape,x_dtype", [((1, 1, 96), F32), ((3, 5, 1027), BF16),
                                           ((3, 1237, 264), BF16), ((2, 1500, 40), F16),
                                           ((2, 301, 4096), BF16), ((2, 150, 8200), F32)])
def test_a_weight_for_each_token(gate, shape, x_dtype):
    """Every row is then a group of its own, whatever the gate, up to more groups than the launch
    has blocks at once and than the sums take in one turn."""
    for post in (True, False):
        parts = reference.make(shape, [x_dtype, BF16, x_dtype, F32, x_dtype], post=post, gate=gate,
                               weight="token", seed=33)
        check(parts, upstream_of(parts, x_dtype), (gate, shape, post), branch_scale=0.3)
