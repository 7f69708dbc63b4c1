"""The rotary norm of heads on the GPU against the 64-bit reference
(tests/rotary_reference.py derives the bounds).

Head sizes lie on both sides of every place where the kernels change: one lane's
pairs (4 or 8), halves that end inside a vector, values that are not turned, the lanes
of a head from 1 to 64.
"""

import itertools
import threading
import warnings

import pytest
import torch
import torch._dynamo.compiled_autograd as compiled_autograd
import torch.utils.checkpoint
from torch.fx.experimental.proxy_tensor import make_fx

import rotary_reference as reference
from gfx1010_kernels import (
    _C,
    _cabi,
    can_use_rms_norm_rotary,
    gated_residual_rms_norm,
    residual_rms_norm,
    rms_norm_rotary,
    rotary_inverse_frequencies,
)
from rms_reference import same_bits

pytestmark = pytest.mark.gpu
EPS = 1e-6
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
CODE = {F32: 0, F16: 1, BF16: 2}
SIZES = [2, 3, 4, 7, 8, 9, 15, 16, 17, 24, 31, 32, 33, 40, 48, 63, 64, 65, 72, 80, 96, 100, 112, 127,
         128, 129, 144, 160, 192, 200, 255, 256]


def call(parts, **options):
    q, k, positions, frequencies, qw, kw = parts
    options.setdefault("implementation", "gfx950")
    return rms_norm_rotary(q, k, positions, frequencies, q_weight=qw, k_weight=kw, eps=EPS,
                           **options)


def step(parts, upstream, **options):
    """Outputs and the gradients of q, k, q_weight and k_weight (None without one)."""
    q, k, positions, frequencies, qw, kw = parts
    leaves = [None if t is None else t.detach().requires_grad_() for t in (q, k, qw, kw)]
    outputs = call((*leaves[:2], positions, frequencies, *leaves[2:]), **options)
    given = [t for t in leaves if t is not None]
    grads = iter(torch.autograd.grad([t for t in outputs if t is not None], given, upstream))
    return outputs, [None if t is None else next(grads) for t in leaves]


def to_gpu(parts):
    return [None if t is None else t.cuda() for t in parts]


def upstream_of(parts, seed=0):
    generator = torch.Generator().manual_seed(seed + 50)
    return [torch.randn(t.shape, generator=generator).to(t.dtype) for t in parts[:2]
            if t is not None]


def check(parts, what, *, sections=None, arrangement="blocks", interleaved=False, seed=0):
    q, k, positions, frequencies, qw, kw = parts
    positions = positions if sections else positions[0]
    parts = (q, k, positions, frequencies, qw, kw)
    angles = reference.angles_of(positions, frequencies, sections, arrangement, q.shape[:-2])
    upstream = upstream_of(parts, seed)
    outputs, grads = step(to_gpu(parts), [t.cuda() for t in upstream], sections=sections,
                          arrangement=arrangement, interleaved=interleaved)
    for i, (heads, weight) in enumerate(((q, qw), (k, kw))):
        if heads is None:
            assert outputs[i] is None
            continue
        reference.check_forward(outputs[i], heads, weight, angles, interleaved, EPS, (what, i))
        reference.check_gradients(grads[i], grads[2 + i], heads, weight, upstream[i], angles,
                                  interleaved, EPS, (what, i))


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("interleaved", [False, True])
def test_sizes(size, interleaved):
    for dtype, norm in ((BF16, True), (F32, True), (F16, False)):
        for pairs in sorted({size // 2, max(1, size // 3), max(1, size // 8), 1}):
            parts = reference.make((2, 3), 3, 2, size, dtype, pairs=pairs, norm=norm, seed=size)
            check(parts, (size, pairs, dtype), interleaved=interleaved)


@pytest.mark.parametrize("dtype,weight_dtype", itertools.product([F32, F16, BF16], repeat=2))
@pytest.mark.parametrize("position_dtype", [torch.int64, torch.int32, torch.float32])
def test_types(dtype, weight_dtype, position_dtype):
    for size in (64, 80):
        q, k, positions, frequencies, qw, kw = reference.make(
            (2, 5), 4, 2, size, dtype, weight_dtype=weight_dtype, position_dtype=position_dtype,
            seed=1)
        if position_dtype == torch.float32:
            positions = positions * 0.37
        for table in (frequencies, frequencies.double() * 1.1):
            check((q, k, positions, table, qw, kw), (size, table.dtype))


@pytest.mark.parametrize("sections", [(16,), (10, 6), (4, 7, 5), (1, 0, 15), (5, 4, 4, 3), (2, 14)])
@pytest.mark.parametrize("arrangement", ["blocks", "cyclic"])
@pytest.mark.parametrize("interleaved", [False, True])
def test_axes(sections, arrangement, interleaved):
    for size in (32, 41):
        parts = reference.make((3, 7), 2, 1, size, F32, pairs=16, axes=len(sections), seed=2)
        check(parts, (sections, size), sections=sections, arrangement=arrangement,
              interleaved=interleaved)


@pytest.mark.parametrize("q_heads,k_heads", [(1, 1), (1, 0), (5, 0), (7, 1), (32, 8), (3, 129)])
@pytest.mark.parametrize("tokens", [(1,), (1, 1), (3,), (2, 1), (70, 1), (1, 33), (2, 2, 5), ()])
def test_heads_and_tokens(q_heads, k_heads, tokens):
    parts = reference.make(tokens, q_heads, k_heads, 64, BF16, seed=3)
    check(parts, (tokens, q_heads, k_heads))


@pytest.mark.parametrize("tokens,size,heads", [(1025, 128, 2), (4100, 64, 3), (2500, 16, 1),
                                               (5000, 256, 1)])
def test_tiles_of_tokens(tokens, size, heads):
    """Token counts on both sides of the sizes of a tile, and more tiles than blocks."""
    for norm in (True, False):
        parts = reference.make((tokens,), heads, 1, size, BF16, norm=norm, seed=tokens)
        check(parts, (tokens, size))


@pytest.mark.parametrize("norms", [(True, False), (False, True)])
def test_one_of_the_two_normed(norms):
    parts = list(reference.make((2, 9), 4, 2, 48, F32, seed=4))
    for i, own in enumerate(norms):
        if not own:
            parts[4 + i] = None
    check(parts, norms)


@pytest.mark.parametrize("far", [1 << 17, 1 << 20, 1 << 24, 1 << 33])
def test_far_positions_keep_their_angles(far):
    """The reference multiplies in 64 bits as well; past 2^27 radians (2^33 positions)
    an angle's own rounding is 2^-20 of one, and frequencies that are powers of two
    keep it exact."""
    parts = list(reference.make((2, 9), 2, 1, 64, F32, norm=False, seed=5, far=far))
    if far > 1 << 27:
        parts[3] = 2.0 ** -torch.arange(32).float()
        assert (parts[2] >= far).all()
    check(parts, far)


def test_a_known_turn():
    q = torch.tensor([[[1.0, 0.0, 5.0, 0.0, 2.0, 7.0]]], device="cuda")
    frequencies = torch.tensor([torch.pi / 2, torch.pi], device="cuda", dtype=torch.float64)
    out, none = rms_norm_rotary(q, None, torch.tensor([1], device="cuda"), frequencies,
                                implementation="gfx950")
    assert none is None
    expected = torch.tensor([[[-5.0, 0.0, 1.0, 0.0, 2.0, 7.0]]])
    assert ((out.cpu() - expected).abs() <= 2.0 ** -21).all()
    zero = rms_norm_rotary(q, None, torch.tensor([0], device="cuda"), frequencies,
                           implementation="gfx950")[0]
    assert same_bits(zero, q)


def layouts(tensor):
    """The same heads [batch, length, heads, size] in other memory."""
    b, n, h, d = tensor.shape
    wide = torch.zeros(b, n, h + 3, d, dtype=tensor.dtype, device="cuda")
    wide[:, :, 2:2 + h] = tensor
    yield "part of a joint projection", wide[:, :, 2:2 + h]
    yield "heads outermost", tensor.permute(2, 0, 1, 3).contiguous().permute(1, 2, 0, 3)
    yield "heads before tokens", tensor.transpose(1, 2).contiguous().transpose(1, 2)
    padded = torch.zeros(b, n, h, d + 3, dtype=tensor.dtype, device="cuda")
    padded[..., 1:1 + d] = tensor
    yield "padded heads, off alignment", padded[..., 1:1 + d]
    yield "values apart", tensor.transpose(2, 3).contiguous().transpose(2, 3)
    yield "tokens backwards", tensor.flip(1).contiguous().flip(1)
    longer = torch.zeros(b, n + 4, h, d, dtype=tensor.dtype, device="cuda")
    longer[:, 1:1 + n] = tensor
    yield "part of longer sequences", longer[:, 1:1 + n]


@pytest.mark.parametrize("size", [64, 80, 37])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_strides_offsets_and_orders(size, dtype):
    parts = to_gpu(reference.make((3, 5), 4, 2, size, dtype, axes=2, seed=6))
    upstream = [t.cuda() for t in upstream_of(parts)]
    options = dict(sections=(size // 2 - 3, 3))
    expected = step(parts, upstream, **options)
    positions = parts[2]
    strided = torch.zeros(3, 2, 5, dtype=positions.dtype, device="cuda").transpose(0, 1)
    strided.copy_(positions)
    weights = [torch.stack([t, t], -1)[..., 1] for t in parts[4:]]
    for (name, q), (_, k), (_, gq), (_, gk) in zip(*map(layouts, [*parts[:2], *upstream])):
        found = step([q, k, strided, parts[3], *weights], [gq, gk], **options)
        for a, b in zip([*found[0], *found[1]], [*expected[0], *expected[1]]):
            assert a.is_contiguous() and same_bits(a, b), name


@pytest.mark.parametrize("shape", [(5,), (1, 5), (3, 1), (1,), (), (3, 5)])
def test_positions_that_broadcast(shape):
    parts = to_gpu(reference.make((3, 5), 2, 1, 32, F32, seed=7))
    positions = torch.randint(0, 99, shape, device="cuda")
    whole = positions.expand(3, 5).contiguous()
    for a, b in zip(call([*parts[:2], positions, *parts[3:]]),
                    call([*parts[:2], whole, *parts[3:]])):
        assert same_bits(a, b)
    axes = torch.stack([positions, positions + 1])
    for a, b in zip(call([*parts[:2], axes, *parts[3:]], sections=(9, 7)),
                    call([*parts[:2], torch.stack([whole, whole + 1]), *parts[3:]],
                         sections=(9, 7))):
        assert same_bits(a, b)


def test_broadcast_heads_get_the_sums_of_their_gradients():
    """One key head read by all queries' groups: a stride of zero."""
    q, k, positions, frequencies, qw, kw = to_gpu(reference.make((2, 5), 4, 1, 32, F32, seed=8))
    leaf = k.detach().requires_grad_()
    out = call([q, leaf.expand(2, 5, 4, 32), positions[0], frequencies, qw, kw])[1]
    (grad,) = torch.autograd.grad(out, leaf, torch.ones_like(out))
    alone = k.detach().requires_grad_()
    (one,) = torch.autograd.grad(call([q, alone, positions[0], frequencies, qw, kw])[1], alone,
                                 torch.ones_like(k))
    assert torch.allclose(grad, 4 * one, rtol=1e-6, atol=1e-6)


def test_dispatch_reaches_the_kernels(recwarn):
    parts = to_gpu(reference.make((2, 5), 4, 2, 32, BF16, seed=9))
    parts[2] = parts[2][0]
    expected = call(parts)
    keywords = dict(q_weight=parts[4], k_weight=parts[5])
    assert can_use_rms_norm_rotary(*parts[:4], **keywords)
    for implementation in ("auto", "gfx1010"):
        for a, b in zip(call(parts, implementation=implementation), expected):
            assert same_bits(a, b)
    assert not recwarn.list
    wide = torch.zeros(2, 1, 258, device="cuda")
    for q, positions, frequencies, message in [
        (wide, torch.zeros(2, device="cuda", dtype=torch.int64), parts[3], "1 to 256 values"),
        (parts[0], parts[2].short(), parts[3], "positions must use"),
        (parts[0], parts[2], parts[3].half(), "inverse_frequencies must"),
        (parts[0], parts[2], parts[3].clone().requires_grad_(), "no gradient"),
    ]:
        with pytest.warns(RuntimeWarning, match=message):
            rms_norm_rotary(q, None, positions, frequencies)
        assert not can_use_rms_norm_rotary(q, None, positions, frequencies)
        with pytest.raises(RuntimeError, match=message):
            rms_norm_rotary(q, None, positions, frequencies, implementation="gfx950")
    with pytest.raises(RuntimeError, match="must be HIP tensors"):
        call([*parts[:2], parts[2].cpu(), *parts[3:]])
    for message, bad in [("sections", dict(sections=(3, 4))), ("broadcast", {})]:
        given = [*parts[:2], parts[2] if bad else parts[2][:, :3], *parts[3:]]
        for implementation in ("auto", "gfx950", "torch"):
            with pytest.raises(ValueError, match=message):
                call(given, implementation=implementation, **bad)


def test_sections_whose_sum_wraps_round():
    """Four sections that add up to the pairs in 64 bits alone are refused."""
    parts = to_gpu(reference.make((5,), 3, 2, 40, F32, axes=4, seed=9))
    pairs = parts[3].shape[0]
    sections = (1 << 62, 1 << 62, 1 << 62, (1 << 62) + pairs)
    for implementation in ("auto", "gfx950", "torch"):
        with pytest.raises(ValueError, match="sections must add up"):
            call(parts, sections=sections, implementation=implementation)
    with pytest.raises(RuntimeError, match="that add up to"):
        _C.rms_norm_rotary(*parts[:4], sections, False, False, *parts[4:], EPS)


@pytest.mark.parametrize("shape", [(0, 4, 32), (2, 0, 4, 32), (2, 3, 0, 32)])
def test_empty(shape):
    q = torch.zeros(shape, device="cuda", requires_grad=True)
    weight = torch.ones(32, device="cuda", requires_grad=True)
    positions = torch.zeros(shape[:-2], device="cuda", dtype=torch.int64)
    frequencies = torch.ones(16, device="cuda")
    k = torch.randn(*shape[:-2], 1, 32, device="cuda", requires_grad=True)
    for key in (None, k):
        out, k_out = rms_norm_rotary(q, key, positions, frequencies, q_weight=weight,
                                     implementation="gfx950")
        assert out.shape == shape and (k_out is None) == (key is None)
        grads = torch.autograd.grad(out.sum() + (0 if key is None else k_out.sum()), [q, weight])
        assert grads[0].shape == shape and grads[1].shape == (32,) and not grads[1].any()


@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("norm", [True, False])
def test_one_output_alone(which, norm):
    parts = to_gpu(reference.make((2, 5), 3, 2, 40, F32, norm=norm, seed=10))
    parts[2] = parts[2][0]
    upstream = [t.cuda() for t in upstream_of(parts)]
    expected = step(parts, upstream)[1]
    leaves = [None if t is None else t.detach().requires_grad_()
              for t in (parts[0], parts[1], parts[4], parts[5])]
    output = call((*leaves[:2], parts[2], parts[3], *leaves[2:]))[which]
    given = [t for t in leaves if t is not None]
    grads = iter(torch.autograd.grad(output, given, upstream[which], allow_unused=True))
    for place, leaf in enumerate(leaves):
        if leaf is None:
            continue
        grad = next(grads)
        assert (grad is None) == (place % 2 != which)
        assert grad is None or same_bits(grad, expected[place])


def test_parts_of_the_gradient():
    parts = to_gpu(reference.make((2, 5), 3, 2, 40, F32, seed=11))
    parts[2] = parts[2][0]
    upstream = [t.cuda() for t in upstream_of(parts)]
    expected = step(parts, upstream)[1]
    for wanted in itertools.chain(itertools.combinations(range(4), 1),
                                  itertools.combinations(range(4), 2)):
        leaves = [t.detach().requires_grad_(i in wanted)
                  for i, t in enumerate((parts[0], parts[1], parts[4], parts[5]))]
        outputs = call((*leaves[:2], parts[2], parts[3], *leaves[2:]))
        grads = torch.autograd.grad(
            [o for o in outputs if o.requires_grad], [leaves[i] for i in wanted],
            [g for o, g in zip(outputs, upstream) if o.requires_grad])
        for grad, place in zip(grads, wanted):
            assert same_bits(grad, expected[place])


def test_gradients_are_those_of_differences():
    """Central differences of the forward itself, in fp32."""
    parts = to_gpu(reference.make((2, 2), 2, 1, 24, F32, seed=12))
    parts[2] = parts[2][0]
    upstream = [t.cuda() for t in upstream_of(parts)]
    grads = step(parts, upstream)[1]
    h = 2.0 ** -6
    for place, index in enumerate((0, 1, 4, 5)):
        direction = torch.randn_like(parts[index])
        direction /= direction.norm()

        def value(sign):
            moved = list(parts)
            moved[index] = parts[index] + sign * h * direction
            return sum((o.double() * g.double()).sum() for o, g in zip(call(moved), upstream))

        slope = (value(1) - value(-1)) / (2 * h)
        along = (grads[place].double() * direction.double()).sum()
        # rounding: 28 u of values near 1 over the step; curvature: the step squared
        assert abs(slope - along) <= 20 * h * h * sum(g.double().norm() for g in upstream)


@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
@pytest.mark.parametrize("norm", [True, False])
def test_heads_that_are_not_finite_stay_alone(bad, norm):
    for size in (16, 72, 128):
        parts = to_gpu(reference.make((2, 9), 5, 2, size, F32, norm=norm, seed=13))
        parts[2] = parts[2][0]
        upstream = [t.cuda() for t in upstream_of(parts)]
        clean = step(parts, upstream)
        parts[0] = parts[0].clone()
        parts[0][1, 2, 3, size // 3] = bad
        upstream[0][0, 4, 1, 2] = bad
        found = step(parts, upstream)
        keep = torch.ones(2, 9, 5, dtype=torch.bool, device="cuda")
        keep[1, 2, 3] = False
        assert same_bits(found[0][0][keep], clean[0][0][keep])
        assert same_bits(found[0][1], clean[0][1])
        assert not found[0][0][1, 2, 3].isfinite().all()
        keep[0, 4, 1] = False
        assert same_bits(found[1][0][keep], clean[1][0][keep])
        assert not found[1][0][0, 4, 1].isfinite().all()
        assert same_bits(found[1][1], clean[1][1])
        if norm:
            assert same_bits(found[1][3], clean[1][3])


@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
@pytest.mark.parametrize("size,pairs", [(48, 8), (80, 16), (41, 5), (128, 32)])
def test_values_that_are_not_turned_stay_alone(bad, size, pairs):
    """Without a norm, a value behind the turned ones is copied, whatever is beside it;
    so is its gradient."""
    for dtype in (F32, BF16):
        parts = to_gpu(reference.make((5,), 3, 1, size, dtype, pairs=pairs, norm=False, seed=28))
        parts[2] = parts[2][0]
        for column in {2 * pairs, size - 1, (2 * pairs + size) // 2}:
            q = parts[0].clone()
            q[1, 2, column] = bad
            for interleaved in (False, True):
                (out, _), grads = step([q, *parts[1:]], [q, parts[1]], interleaved=interleaved)
                for found in (out, grads[0]):
                    assert same_bits(found[..., 2 * pairs:], q[..., 2 * pairs:])
                    assert found[..., :2 * pairs].isfinite().all()


def test_positions_that_are_not_finite_stay_in_their_token():
    parts = to_gpu(reference.make((6,), 3, 1, 32, F32, seed=14, position_dtype=torch.float32))
    positions = parts[2][0].clone()
    clean = call([*parts[:2], positions, *parts[3:]])
    positions[2], positions[4] = float("inf"), float("nan")
    found = call([*parts[:2], positions, *parts[3:]])
    for a, b in zip(found, clean):
        assert a[[2, 4]].isnan().all() and same_bits(a[[0, 1, 3, 5]], b[[0, 1, 3, 5]])


# The graph, threads, streams, buffers.

def test_sums_are_the_same_on_every_run():
    parts = to_gpu(reference.make((4, 700), 8, 2, 128, BF16, seed=15))
    parts[2] = parts[2][0]
    upstream = [t.cuda() for t in upstream_of(parts)]
    first = step(parts, upstream)[1]
    for _ in range(3):
        assert all(same_bits(a, b) for a, b in zip(step(parts, upstream)[1], first))


@pytest.mark.parametrize("norm", [True, False])
def test_the_graph_is_kept_and_released_as_any(norm):
    parts = to_gpu(reference.make((2, 5), 3, 2, 40, F32, norm=norm, seed=16))
    leaves = [t.requires_grad_() for t in (parts[0], parts[1], parts[4], parts[5]) if t is not None]

    def forward():
        q, k = call([*parts[:2], parts[2][0], *parts[3:]])
        return q.square().sum() + k.sin().sum()

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
    parts = to_gpu(reference.make((5,), 3, 2, 40, F32, seed=17))
    parts[0].requires_grad_()
    q = call([*parts[:2], parts[2][0], *parts[3:]])[0]
    (grad,) = torch.autograd.grad(q.square().sum(), parts[0], create_graph=True)
    with pytest.raises(RuntimeError, match="second-order gradients"):
        grad.square().sum().backward()


def test_what_is_kept():
    """Heads are kept, and may not change, only where they are normed."""
    for norm in (True, False):
        q, _, positions, frequencies, qw, _ = to_gpu(reference.make((5,), 3, 0, 40, F32, norm=norm,
                                                                    seed=18))
        leaf = q.clone().requires_grad_()
        heads = leaf * 1.0
        out = rms_norm_rotary(heads, None, positions[0], frequencies, q_weight=qw)[0]
        heads.add_(1.0)
        if norm:
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                out.sum().backward()
        else:
            out.sum().backward()


def test_forward_mode_takes_the_torch_path():
    parts = to_gpu(reference.make((5,), 3, 2, 40, F32, seed=19))
    parts[2] = parts[2][0]
    with torch.autograd.forward_ad.dual_level():
        parts[0] = torch.autograd.forward_ad.make_dual(parts[0], torch.ones_like(parts[0]))
        with pytest.warns(RuntimeWarning, match="forward-mode"):
            q = call(parts, implementation="auto")[0]
        assert torch.autograd.forward_ad.unpack_dual(q).tangent is not None
        with pytest.raises(RuntimeError, match="forward-mode"):
            call(parts)


def test_two_threads_at_once():
    cases = []
    for size in (64, 128):
        parts = to_gpu(reference.make((3, 129), 8, 2, size, BF16, seed=size))
        parts[2] = parts[2][0]
        cases.append((parts, [t.cuda() for t in upstream_of(parts)]))

    def work(parts, upstream):
        outputs, grads = step(parts, upstream)
        return [*outputs, *grads]

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
    parts = to_gpu(reference.make((4, 512), 8, 2, 128, BF16, seed=20))
    parts[2] = parts[2][0]
    upstream = [t.cuda() for t in upstream_of(parts)]
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


@pytest.mark.parametrize("size", [2, 3, 16, 37, 64, 80, 128, 129, 255, 256])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("interleaved", [0, 1])
def test_nothing_is_written_outside_the_outputs(size, dtype, interleaved):
    tokens, counts, code = 7, (3, 2), CODE[dtype]
    stream = torch.cuda.current_stream().cuda_stream
    library = _cabi.library()
    for pairs in sorted({size // 2, max(1, size // 3)}):
        q, k, positions, frequencies, qw, kw = to_gpu(
            reference.make((tokens,), *counts, size, dtype, pairs=pairs, seed=size))
        grads = [torch.randn_like(t) for t in (q, k)]
        table = _cabi.RlnRotary(positions.data_ptr(), 0, tokens, 0, 1, frequencies.data_ptr(), 0,
                                None, 1, pairs, interleaved)
        checks, made = [], []

        def sides(backward):
            for heads, grad, weight in ((q, grads[0], qw), (k, grads[1], kw)):
                out, verify = guarded(heads.numel(), dtype)
                sums, verify_sums = guarded(size, dtype)
                checks.extend([verify, verify_sums])
                made.extend([out.view(heads.shape), sums] if backward else [out.view(heads.shape)])
                count = heads.shape[1]
                yield _cabi.RlnRotarySide(
                    _cabi.RlnHeads(heads.data_ptr(), 0, count * size, size),
                    _cabi.RlnHeads(grad.data_ptr(), 0, count * size, size), count,
                    weight.data_ptr(), code, out.data_ptr(), sums.data_ptr() if backward else None)

        assert library.rln_rotary_forward(*sides(False), code, table, 1, tokens, size, EPS,
                                          stream) == 0
        bytes_ = library.rln_rotary_backward_workspace_bytes(1, tokens, *counts, size, pairs, code)
        workspace, verify = guarded(bytes_, torch.uint8)
        checks.append(verify)
        assert library.rln_rotary_backward(*sides(True), code, table, 1, tokens, size, EPS,
                                           workspace.data_ptr(), bytes_, stream) == 0
        torch.cuda.synchronize()
        for verify in checks:
            verify()
        outputs, found = step([q, k, positions[0], frequencies, qw, kw], grads,
                              interleaved=bool(interleaved))
        for a, b in zip(made, [*outputs, found[0], found[2], found[1], found[3]]):
            assert same_bits(a, b)


# Graphs, compilation, traces.

def test_captured_steps_replay():
    """Two captured training steps that share the allocator's graph pool, and a
    captured serving call, replayed several times with new inputs and positions."""
    parts = to_gpu(reference.make((3, 50), 6, 2, 72, F32, axes=2, seed=21))
    upstream = [t.cuda() for t in upstream_of(parts)]
    leaves = [t.clone().requires_grad_() for t in (parts[0], parts[1], parts[4], parts[5])]
    positions = parts[2].clone()
    options = dict(sections=(20, 16), interleaved=True, implementation="auto")

    def work(leaves, positions):
        outputs = call((*leaves[:2], positions, parts[3], *leaves[2:]), **options)
        with torch.no_grad():
            served = call((*leaves[:2], positions, parts[3], *leaves[2:]), **options)
        return [*outputs, *served, *torch.autograd.grad(outputs, leaves, upstream)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work(leaves, positions)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outputs, pool = [], [], None
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=pool):
            outputs.append(work(leaves, positions))
        pool = graph.pool()
        graphs.append(graph)
    for turn in range(4):
        fresh = [t.detach() + 0.25 * turn for t in (parts[0], parts[1], parts[4], parts[5])]
        with torch.no_grad():
            for leaf, value in zip(leaves, fresh):
                leaf.copy_(value)
            positions.copy_(parts[2] + turn)
        expected = work([t.clone().requires_grad_() for t in fresh], parts[2] + turn)
        for graph, found in zip(graphs, outputs):
            graph.replay()
            torch.cuda.synchronize()
            assert all(same_bits(a, b) for a, b in zip(found, expected)), turn


@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("k_heads", [2, 0])
def test_compiled_step_equals_the_eager_one(norm, k_heads):
    parts = to_gpu(reference.make((2, 9), 4, k_heads, 48, BF16, norm=norm, axes=2, seed=22))
    given = [t for t in (parts[0], parts[1], parts[4], parts[5]) if t is not None]
    upstream = [t.cuda() for t in upstream_of(parts)]

    def forward(*leaves):
        it = iter(leaves)
        q, k, qw, kw = (None if t is None else next(it)
                        for t in (parts[0], parts[1], parts[4], parts[5]))
        return tuple(t for t in call((q, k, parts[2], parts[3], qw, kw), sections=(16, 8),
                                     implementation="auto") if t is not None)

    results = []
    for function in (forward, torch.compile(forward, backend="aot_eager", fullgraph=True)):
        leaves = [t.clone().requires_grad_() for t in given]
        outputs = function(*leaves)
        results.append([*outputs, *torch.autograd.grad(outputs, leaves, upstream)])
    for a, b in zip(*results):
        assert same_bits(a, b)
    grads = []
    for function in (forward, torch.compile(forward, backend="aot_eager", fullgraph=True)):
        leaves = [t.clone().requires_grad_(i == 0) for i, t in enumerate(given)]
        grads.append(torch.autograd.grad(function(*leaves)[0], leaves[0], upstream[0])[0])
    assert same_bits(*grads)


@pytest.mark.parametrize("implementation", ["auto", "gfx950", "torch"])
def test_traces_hold_the_operator(implementation):
    parts = to_gpu(reference.make((2, 4), 3, 1, 32, F32, seed=23))
    parts[2] = parts[2][0]
    call(parts)

    def function(*given):
        return call(given, implementation=implementation)

    fresh = [parts[0] + 0.5, parts[1] - 1.0, parts[2] + 7, *parts[3:]]
    # TorchScript's fuser contracts products and sums of the PyTorch path: two results,
    # each within 28 u of |n1| + |n2|, normed values of at most sqrt(32) times a weight.
    largest = 32 ** 0.5 * max(float(t.abs().max()) for t in parts[4:])
    tolerance = 2 * 28 * 2.0 ** -24 * 2 * largest
    with torch.no_grad(), warnings.catch_warnings():
        warnings.simplefilter("ignore")
        for graph in (torch.jit.trace(function, parts), make_fx(function)(*parts)):
            for given in (parts, fresh):
                for a, b in zip(graph(*given), function(*given)):
                    assert (same_bits(a, b) if implementation != "torch"
                            else ((a - b).abs() <= tolerance).all())
    with pytest.raises(RuntimeError, match="recorded into a graph"):
        make_fx(lambda q, k, p, f, a, b: _C.rms_norm_rotary(q, k, p, f, [], False, False, a, b,
                                                            EPS))(*parts)


@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("sections", [(12, 8), (4, 16)])
def test_compiled_autograd(norm, sections):
    def grads(seed, backend):
        torch._dynamo.reset()
        parts = to_gpu(reference.make((2, 6), 4, 2, 40, F32, norm=norm, axes=2, seed=seed))
        leaves = [t.requires_grad_() for t in (parts[0], parts[1], parts[4], parts[5])
                  if t is not None]
        q, k = call(parts, sections=sections, implementation="auto")
        loss = q.sin().sum() + k.square().sum()
        if backend is None:
            loss.backward()
        else:
            with compiled_autograd._enable(torch.compile(backend=backend)):
                loss.backward()
        return [t.grad for t in leaves]

    for seed in (0, 1):
        for backend in ("eager", "aot_eager"):
            for a, b in zip(grads(seed, backend), grads(seed, None)):
                assert same_bits(a, b)


def test_compiled_autograd_tells_calls_apart():
    """Backwards that differ in constants alone, one after the other."""
    q, k, positions, frequencies, qw, kw = to_gpu(reference.make((2, 6), 4, 2, 40, F32, axes=2,
                                                                 seed=24))

    def grads(sections, interleaved, enabled):
        leaf = q.detach().requires_grad_()
        out = call([leaf, k, positions, frequencies, qw, kw], sections=sections,
                   interleaved=interleaved)[0]
        if not enabled:
            out.sin().sum().backward()
        else:
            with compiled_autograd._enable(torch.compile(backend="eager")):
                out.sin().sum().backward()
        return leaf.grad

    torch._dynamo.reset()
    for options in (((12, 8), False), ((12, 8), True), ((8, 12), True), ((12, 8), False)):
        assert same_bits(grads(*options, True), grads(*options, False))


def test_transforms_and_fake_tensors_are_refused():
    from torch._subclasses.fake_tensor import FakeTensorMode

    parts = to_gpu(reference.make((5,), 3, 2, 40, F32, seed=25))
    parts[2] = parts[2][0]
    expected = call(parts)
    with pytest.raises(Exception):
        torch.func.grad(lambda t: call([t, *parts[1:]])[0].sum())(parts[0])
    with FakeTensorMode(allow_non_fake_inputs=True), pytest.raises(Exception):
        call(parts)
    for a, b in zip(call(parts), expected):
        assert same_bits(a, b)


def test_heads_past_two_to_the_31_elements():
    """Offsets of the last tokens pass 2^31 elements (and 2^32 bytes)."""
    tokens, heads, size = (1 << 31) // (64 * 256) + 3, 64, 256
    q, _, positions, frequencies, qw, _ = reference.make((1,), heads, 0, size, BF16, seed=26,
                                                         far=1000)
    whole = torch.zeros(tokens, heads, size, device="cuda", dtype=BF16)
    whole[-1] = q[0]
    weight = qw.cuda().requires_grad_()
    whole.requires_grad_()
    at = torch.zeros(tokens, device="cuda", dtype=torch.int64)
    at[-1] = positions[0, 0]
    out = rms_norm_rotary(whole, None, at, frequencies.cuda(), q_weight=weight, eps=EPS,
                          implementation="gfx950")[0]
    angles = reference.angles_of(positions[0], frequencies, None, "blocks", (1,))
    reference.check_forward(out[-1:], q, qw, angles, False, EPS, "last token")
    assert not out[:-1].any()
    upstream = torch.zeros_like(out)
    upstream[-1] = 1.0
    grads = torch.autograd.grad(out, [whole, weight], upstream)
    assert not grads[0][:-1].any()
    reference.check_gradients(grads[0][-1:], grads[1], q, qw, torch.ones_like(q), angles, False,
                              EPS, "last token")


# Together, as they are used.

class Attention(torch.nn.Module):
    """Grouped heads with norms of their own and positions of three axes; the
    products and the softmax in fp32."""

    def __init__(self, hidden, heads, groups, size, implementation):
        super().__init__()
        self.counts, self.size = (heads, groups, groups), size
        self.joint = torch.nn.Linear(hidden, (heads + 2 * groups) * size, bias=False)
        self.q_norm, self.k_norm = (torch.nn.Parameter(1 + 0.1 * torch.randn(size))
                                    for _ in range(2))
        self.out = torch.nn.Linear(heads * size, hidden, bias=False)
        self.register_buffer("frequencies", rotary_inverse_frequencies((size // 2,)))
        self.implementation = implementation
        self.positions = None

    def forward(self, x):
        parts = self.joint(x).unflatten(-1, (-1, self.size)).split(self.counts, -2)
        pairs = self.size // 2
        q, k = rms_norm_rotary(parts[0], parts[1], self.positions, self.frequencies,
                               sections=(pairs - 8, 4, 4), q_weight=self.q_norm,
                               k_weight=self.k_norm, implementation=self.implementation)
        heads, groups, _ = self.counts
        q, k, v = (t.transpose(1, 2).float() for t in (q, k, parts[2]))
        k, v = (t.repeat_interleave(heads // groups, 1) for t in (k, v))
        scores = q @ k.transpose(-1, -2).contiguous() / self.size ** 0.5
        mask = torch.ones(scores.shape[-2:], dtype=torch.bool, device=x.device).triu(1)
        weights = scores.masked_fill(mask, float("-inf")).softmax(-1)
        return self.out((weights @ v).transpose(1, 2).flatten(-2).to(x.dtype))


class Block(torch.nn.Module):
    def __init__(self, hidden, implementation):
        super().__init__()
        self.ln_1, self.ln_2 = torch.nn.RMSNorm(hidden, eps=EPS), torch.nn.RMSNorm(hidden, eps=EPS)
        self.post_1 = torch.nn.RMSNorm(hidden, eps=EPS)
        self.attn = Attention(hidden, 6, 2, 32, implementation)
        self.mlp = torch.nn.Sequential(torch.nn.Linear(hidden, 2 * hidden), torch.nn.SiLU(),
                                       torch.nn.Linear(2 * hidden, hidden))
        self.gate = torch.nn.Parameter(torch.randn(hidden))


@pytest.mark.parametrize("training", [True, False])
def test_a_stack_of_blocks(training):
    """Gated pre-norm blocks around attention with turned heads: the kernels against
    the PyTorch path of the same operators in the same model, in fp32."""
    from gfx1010_kernels import prenorm_forward

    results = []
    for implementation in ("gfx950", "torch"):
        torch.manual_seed(27)
        blocks = torch.nn.ModuleList(Block(192, implementation) for _ in range(3)).cuda()
        final = torch.nn.RMSNorm(192, eps=EPS).cuda()
        x = torch.randn(2, 40, 192, device="cuda", requires_grad=True)
        for block in blocks:
            block.attn.positions = torch.randint(
                0, 500, (3, 2, 40), device="cuda", generator=torch.Generator("cuda").manual_seed(1))
        with torch.set_grad_enabled(training):
            stream, out = prenorm_forward(
                x, blocks, final, post_ln1="post_1", gate1="gate",
                gate2=lambda block: block.gate.tanh(), branch_scale=0.5,
                implementation=implementation)
            found = [stream, out]
            if training:
                leaves = [x, *(p for p in [*blocks.parameters(), *final.parameters()]
                               if p.requires_grad)]
                found += torch.autograd.grad((stream.sin() + out * out).sum(), leaves,
                                             allow_unused=True)
        results.append(found)
    for a, b in zip(*results):
        assert (a is None) == (b is None)
        if a is not None:
            # Sums of a few hundred fp32 terms through six sublayers.
            assert (a - b).abs().max() <= 2e-4 * b.abs().max()


def test_the_norms_of_a_block_agree():
    """The first norm of a stack and the gated one that follows, on one stream."""
    x = torch.randn(4, 96, device="cuda")
    weight = torch.rand(96, device="cuda")
    first = residual_rms_norm(x, None, weight, EPS)[1]
    second = gated_residual_rms_norm(x, torch.zeros_like(x), weight, EPS, branch_weight=weight)[1]
    assert same_bits(first, second)


# Tables that require a gradient.

@pytest.mark.parametrize("table", [2, 3])
@pytest.mark.parametrize("implementation", ["gfx950", "gfx1010"])
def test_graphs_drop_no_gradient_of_the_tables(table, implementation):
    """Positions or frequencies that require a gradient are refused where they would lose it, in
    every way to the registered operator."""
    parts = to_gpu(reference.make((2, 5), 4, 2, 32, F32, position_dtype=F32, seed=27))
    parts[2] = parts[2][0]
    plain = list(parts)
    parts[table] = parts[table].clone().requires_grad_()

    def function(*given):
        return call(given, implementation=implementation)

    refused = "positions and inverse_frequencies have no gradient"
    for fullgraph in (False, True):
        torch._dynamo.reset()
        with pytest.raises(RuntimeError, match=refused):
            torch.compile(function, backend="aot_eager", fullgraph=fullgraph)(*parts)
    with pytest.raises(RuntimeError, match=refused):
        make_fx(function)(*parts)
    operator = torch.ops.gfx1010_kernels.rotary_forward
    with pytest.raises(RuntimeError, match=refused):
        operator(*parts[:4], [], False, False, *parts[4:], EPS)
    with warnings.catch_warnings(), torch.no_grad():
        warnings.simplefilter("ignore")
        traced = torch.jit.trace(function, plain)
        expected = call(parts)
        for found in (operator(*parts[:4], [], False, False, *parts[4:], EPS), traced(*parts)):
            assert all(same_bits(a, b) for a, b in zip(found, expected))
    with warnings.catch_warnings():
        warnings.simplefilter("ignore")
        with pytest.raises(RuntimeError, match=refused):
            torch.jit.trace(function, parts, check_trace=False)
    with pytest.raises(RuntimeError, match=refused):
        traced(*parts)


@pytest.mark.parametrize("table", [2, 3])
def test_compiled_auto_calls_differentiate_the_tables(table):
    """A gradient is a sum of upstream (a cosine) * turned value * the other table over heads and
    tokens or pairs, S = |n1| + |n2| bounding the turned values. A term carries 28 u of the norm and
    the turn, as much times S through the cosine, and 8 u of its own products; the sum adds its
    number of terms. Both runs are that near to the formula's value."""
    parts = to_gpu(reference.make((2, 5), 4, 2, 32, F32, position_dtype=F32, seed=27))
    parts[2] = parts[2][0] % 7

    def function(*given):
        q, k = call(given, implementation="auto")
        return q.sin().sum() + k.sin().sum()

    grads = []
    for run in (function, torch.compile(function, backend="aot_eager", fullgraph=True)):
        torch._dynamo.reset()
        given = list(parts)
        given[table] = given[table].clone().requires_grad_()
        with warnings.catch_warnings():
            warnings.simplefilter("ignore")  # the PyTorch path says that it is taken
            grads.append(torch.autograd.grad(run(*given), given[table])[0].double())
    size = torch.cat([reference.pair_size(
        heads.double() * reference.rstd_of(heads.double(), EPS) * weight.double(), 16, False)
        for heads, weight in ((parts[0], parts[4]), (parts[1], parts[5]))], 2)
    other = parts[3].double() if table == 2 else parts[2].double()[..., None]
    over = (2, 3) if table == 2 else (0, 1, 2)  # both values of a pair among the terms
    sums = (size * (other.repeat(2) if table == 2 else other[..., None]).abs()).sum(over)
    sums = sums if table == 2 else sums[:16] + sums[16:]
    bound = 2 * (36 + 28 * size.max() + size.numel()) * 2.0 ** -24 * sums
    assert grads[0].any()
    assert ((grads[0] - grads[1]).abs() <= bound).all()


def test_sections_are_any_sequence_of_whole_numbers():
    """In every mode, on the first call and on later ones."""
    from test_rotary import sections_of_every_kind

    parts = to_gpu(reference.make((2, 5), 4, 2, 32, F32, axes=2, seed=28))
    keywords = dict(q_weight=parts[4], k_weight=parts[5])
    expected = call(parts, sections=(9, 7))
    for implementation in ("auto", "gfx950", "gfx1010"):
        for sections in sections_of_every_kind((9, 7)):
            found = call(parts, sections=sections, implementation=implementation)
            assert all(same_bits(a, b) for a, b in zip(found, expected)), type(sections)
            assert can_use_rms_norm_rotary(*parts[:4], sections=sections, **keywords)
    for sections in ((9.5, 6.5), torch.tensor([9.5, 6.5])):
        for implementation in ("auto", "gfx950", "torch"):
            with pytest.raises(ValueError, match="whole numbers"):
                call(parts, sections=sections, implementation=implementation)
        assert not can_use_rms_norm_rotary(*parts[:4], sections=sections, **keywords)


def test_what_transforms_and_fake_tensors_are_refused_for():
    """The kernels ask for addresses, which a transform's tensor does not have and a fake output's
    are null."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    parts = to_gpu(reference.make((2, 5), 4, 2, 32, F32, seed=25))
    parts[2] = parts[2][0]
    call(parts, implementation="auto")
    for implementation in ("auto", "gfx950"):
        options = dict(implementation=implementation)
        with pytest.raises(RuntimeError, match="data pointer"):
            torch.func.grad(lambda t: call([t, *parts[1:]], **options)[0].sum())(parts[0])
        with pytest.raises(RuntimeError, match="data pointer"):
            torch.func.vmap(lambda q, k, p: call([q, k, p, *parts[3:]], **options)[0])(*parts[:3])
        with FakeTensorMode(allow_non_fake_inputs=True), pytest.raises(
                RuntimeError, match="must not be null|data is not allocated"):
            call(parts, **options)
        assert call(parts, **options)[0].isfinite().all()


# Tokens that are no single run: positions shared by the samples, heads before tokens.

@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("dtype,size,interleaved", [(BF16, 128, False), (F16, 72, True),
                                                    (F32, 37, False)])
@pytest.mark.parametrize("tokens", [(3, 1), (3, 37), (1, 401), (2, 1283), (2, 3, 130)])
def test_shared_positions_are_those_of_each_sample(norm, dtype, size, interleaved, tokens):
    """A step with positions that repeat over the samples against one with positions of their own,
    bit for bit but for the weights' sums, whose order may differ: those against the reference. The
    longest fill several tiles and more than one per block."""
    parts = reference.make(tokens, 3, 2, size, dtype, norm=norm, axes=2, seed=29)
    options = dict(sections=(size // 2 - 4, 4), interleaved=interleaved)
    shared = parts[2].reshape(2, -1, tokens[-1])[:, 0]
    whole = shared.reshape(2, *[1] * (len(tokens) - 1), -1).expand(2, *tokens).contiguous()
    upstream = upstream_of(parts, 29)
    found, expected = (
        step(to_gpu([*parts[:2], positions, *parts[3:]]), [t.cuda() for t in upstream], **options)
        for positions in (shared, whole))
    for a, b in zip([*found[0], *found[1][:2]], [*expected[0], *expected[1][:2]]):
        assert same_bits(a, b)
    angles = reference.angles_of(shared, parts[3], options["sections"], "blocks", tokens)
    for i in range(2):
        reference.check_gradients(None, found[1][2 + i], parts[i], parts[4 + i], upstream[i],
                                  angles, interleaved, EPS, i)


@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("dtype,size", [(BF16, 128), (F16, 64), (F32, 80)])
@pytest.mark.parametrize("tokens", [(1, 1), (4, 1), (3, 37), (2, 1283)])
def test_heads_before_tokens(norm, dtype, size, tokens):
    """[batch, heads, length, size] seen as [batch, length, heads, size], both ways, with positions
    of each sample and shared ones."""
    parts = to_gpu(reference.make(tokens, 3, 2, size, dtype, norm=norm, seed=30))
    upstream = [t.cuda() for t in upstream_of(parts, 30)]

    def turned(heads):
        return heads.transpose(1, 2).contiguous().transpose(1, 2)

    for positions in (parts[2][0], parts[2][0, 0], parts[2][0, :1]):
        given = [*parts[:2], positions, *parts[3:]]
        expected = step(given, upstream)
        found = step([*map(turned, given[:2]), *given[2:]], [turned(t) for t in upstream])
        for a, b in zip([*found[0], *found[1][:2]], [*expected[0], *expected[1][:2]]):
            assert same_bits(a, b)
        angles = reference.angles_of(positions, parts[3], None, "blocks", tokens)
        for i in range(2):
            reference.check_gradients(None, found[1][2 + i], parts[i], parts[4 + i], upstream[i],
                                      angles, False, EPS, i)
