"""The rotary norm of heads on the CPU: the PyTorch path against the reference, the
reference's gradients against differences, dispatch, and refusals."""

import ctypes
import math
import warnings

import pytest
import torch

import rotary_reference as reference
from gfx1010_kernels import (
    _C,
    _cabi,
    can_use_rms_norm_rotary,
    rms_norm_rotary,
    rotary,
    rotary_inverse_frequencies,
)

EPS = 1e-6
F64 = torch.float64
SECTIONS = {1: None, 2: (5, 3), 3: (4, 1, 3), 4: (2, 3, 2, 1)}


def test_angles_of_the_table():
    shared = rotary_inverse_frequencies((2, 6), 100.0)
    assert torch.allclose(shared, torch.tensor([100.0 ** (-i / 8) for i in range(8)], dtype=F64))
    own = rotary_inverse_frequencies((2, 6), 100.0, shared=False, dtype=torch.float32)
    expected = [100.0 ** (-i / 2) for i in range(2)] + [100.0 ** (-i / 6) for i in range(6)]
    assert own.dtype == torch.float32 and torch.allclose(own, torch.tensor(expected))
    for bad in ((), (0,), (3, -1)):
        with pytest.raises(ValueError, match="sections"):
            rotary_inverse_frequencies(bad)


def test_axes_of_pairs():
    assert rotary.axis_of_pairs((2, 1, 3)) == [0, 0, 1, 2, 2, 2]
    assert rotary.axis_of_pairs((4, 2, 2), "cyclic") == [0, 1, 2, 0, 1, 2, 0, 0]
    assert rotary.axis_of_pairs((1, 4), "cyclic") == [0, 1, 0, 1, 0]  # as far as there are pairs
    for sections in SECTIONS.values():
        for arrangement in ("blocks", "cyclic"):
            if sections is not None:
                assert rotary.axis_of_pairs(sections, arrangement) == reference.axes_of(
                    sections, arrangement)


@pytest.mark.parametrize("axes", SECTIONS)
@pytest.mark.parametrize("arrangement", ["blocks", "cyclic"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("norm", [False, True])
def test_torch_path_and_its_gradients_are_the_reference(axes, arrangement, interleaved, norm):
    q, k, positions, frequencies, qw, kw = reference.make((2, 3), 3, 2, 19, F64, pairs=8,
                                                          axes=axes, norm=norm, seed=axes)
    sections = SECTIONS[axes]
    positions = positions if sections else positions[0]
    angles = reference.angles_of(positions, frequencies, sections, arrangement, (2, 3))
    leaves = [t.requires_grad_() for t in (q, k, qw, kw) if t is not None]

    def run(q, k, qw=None, kw=None):
        return rms_norm_rotary(q, k, positions, frequencies, sections=sections,
                               arrangement=arrangement, interleaved=interleaved, q_weight=qw,
                               k_weight=kw, eps=EPS, implementation="torch")

    outputs = run(*leaves)
    upstream = [torch.randn_like(t) for t in outputs]
    grads = torch.autograd.grad(outputs, leaves, upstream)
    for i, (heads, weight) in enumerate(((q, qw), (k, kw))):
        value = heads
        if weight is not None:
            value = heads * reference.rstd_of(heads, EPS) * weight
        assert torch.allclose(outputs[i], reference.turn(value, angles, interleaved), atol=1e-12)
        one, two = reference.gradients(heads, weight, upstream[i], angles, interleaved, EPS)
        assert torch.allclose(grads[i], one[0], atol=1e-12)
        if norm:
            assert torch.allclose(grads[2 + i], two[0], atol=1e-11)
    assert torch.autograd.gradcheck(run, leaves)


def test_known_turns():
    q = torch.tensor([[[1.0, 0.0, 5.0, 0.0, 2.0, 7.0]]], dtype=F64)
    frequencies = torch.tensor([math.pi / 2, math.pi], dtype=F64)
    out = rms_norm_rotary(q, None, torch.tensor([1]), frequencies, implementation="torch")
    assert out[1] is None
    expected = torch.tensor([[[-5.0, 0.0, 1.0, 0.0, 2.0, 7.0]]], dtype=F64)
    assert torch.allclose(out[0], expected, atol=1e-12)
    out = rms_norm_rotary(q, None, torch.tensor([1]), frequencies, interleaved=True,
                          implementation="torch")[0]
    expected = torch.tensor([[[0.0, 1.0, -5.0, 0.0, 2.0, 7.0]]], dtype=F64)
    assert torch.allclose(out, expected, atol=1e-12)


@pytest.mark.parametrize("shape", [(4,), (3, 4), (1, 4), (2, 3, 4), (2, 1, 4), (1,), ()])
def test_positions_broadcast_over_the_tokens(shape):
    q, k, _, frequencies, _, _ = reference.make((2, 3, 4), 2, 1, 8, F64, norm=False)
    for axes in (None, 2):
        positions = torch.randint(0, 50, shape if axes is None else (axes, *shape))
        sections = None if axes is None else (3, 1)
        whole = positions.expand((2, 3, 4)) if axes is None else torch.stack(
            [axis.expand(2, 3, 4) for axis in positions])
        for a, b in zip(*(rms_norm_rotary(q, k, p, frequencies, sections=sections,
                                          implementation="torch") for p in (positions, whole))):
            assert torch.equal(a, b)


def test_positions_may_have_a_gradient_on_the_torch_path():
    q, _, positions, frequencies, _, _ = reference.make((3,), 1, 0, 8, F64, norm=False)
    positions, frequencies = positions[0].double().requires_grad_(), frequencies.requires_grad_()
    with pytest.warns(RuntimeWarning):
        out = rms_norm_rotary(q, None, positions, frequencies)[0]
    assert all(g.any() for g in torch.autograd.grad(out.square().sin().sum(),
                                                    [positions, frequencies]))


# Dispatch and refusals.

def inputs():
    q, k, positions, frequencies, qw, kw = reference.make((2, 3), 4, 2, 16, torch.float32)
    return dict(q=q, k=k, positions=positions[0], inverse_frequencies=frequencies, q_weight=qw,
                k_weight=kw)


def test_auto_falls_back_with_a_warning_and_strict_modes_raise():
    with pytest.warns(RuntimeWarning, match="rotary RMSNorm was not used: all tensors must be HIP tensors"):
        rms_norm_rotary(**inputs())
    assert not can_use_rms_norm_rotary(**inputs())
    for implementation in ("gfx950", "gfx1010"):
        with pytest.raises(RuntimeError, match="must be HIP tensors"):
            rms_norm_rotary(**inputs(), implementation=implementation)
    with pytest.raises(RuntimeError, match="Triton backend"):
        rms_norm_rotary(**inputs(), implementation="triton")
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        rms_norm_rotary(**inputs(), implementation="torch")


@pytest.mark.parametrize("changes,message", [
    (dict(arrangement="turns"), "arrangement"),
    (dict(q=torch.zeros(16)), "dimensions"),
    (dict(k=torch.zeros(2, 4, 2, 16)), "same tokens"),
    (dict(k=torch.zeros(2, 3, 2, 8)), "same tokens"),
    (dict(k=torch.zeros(2, 3, 2, 16).half()), "type"),
    (dict(k=None), "k_weight needs k"),
    (dict(q_weight=torch.zeros(8)), "must match the head size"),
    (dict(inverse_frequencies=torch.zeros(9)), "size / 2"),
    (dict(inverse_frequencies=torch.zeros(0)), "size / 2"),
    (dict(inverse_frequencies=torch.zeros(2, 4)), "size / 2"),
    (dict(sections=(4, 3)), "add up"),
    (dict(sections=(9, -1)), "add up"),
    (dict(sections=()), "at least one"),
    (dict(sections=(4, 2, 2)), "one row for each section"),
    (dict(positions=torch.zeros(3, 2, dtype=torch.long)), "broadcast"),
    (dict(positions=torch.zeros(1, 2, 3, dtype=torch.long)), "broadcast"),
    (dict(sections=(8,), positions=torch.zeros(1, 4, dtype=torch.long)), "broadcast"),
])
def test_argument_checks(changes, message):
    for implementation in ("auto", "torch"):
        with pytest.raises(ValueError, match=message):
            rms_norm_rotary(**dict(inputs(), **changes), implementation=implementation)


def test_reasons():
    class Device:
        def __init__(self, shape, dtype=torch.float32, device=0):
            self.is_cuda, self.device = True, torch.device("cuda", device)
            self.shape, self.ndim, self.dtype = torch.Size(shape), len(shape), dtype
            self.requires_grad = False

    def reason(sections=None, eps=EPS, **changes):
        parts = dict(q=Device((2, 3, 4, 16)), k=Device((2, 3, 2, 16)),
                     positions=Device((3,), torch.int32), frequencies=Device((8,)),
                     q_weight=Device((16,)), k_weight=None)
        parts.update(changes)
        q, k, positions, frequencies, qw, kw = parts.values()
        return rotary._input_reason(q, k, positions, frequencies, sections, qw, kw, eps)

    assert reason() is None and reason(k=None) is None
    for text, changes in [
        ("same HIP device", dict(frequencies=Device((8,), device=1))),
        ("1 to 256", dict(q=Device((2, 3, 4, 257)))),
        ("1 to 256", dict(q=Device((2, 3, 4, 0)))),
        ("must use float16", dict(k=Device((2, 3, 2, 16), F64))),
        ("must use float16", dict(q_weight=Device((16,), F64))),
        ("65536 heads", dict(q=Device((1, 65537, 16)))),
        ("inverse_frequencies must use", dict(frequencies=Device((8,), torch.float16))),
        ("positions must use", dict(positions=Device((3,), torch.int16))),
        ("axes", dict(sections=(2, 2, 2, 1, 1))),
        ("too many tokens", dict(q=Device((1 << 30, 1, 16)))),
        ("eps", dict(eps=-1.0)),
    ]:
        assert text in reason(**changes), changes


def test_the_extension_declines_host_tensors():
    given = inputs()
    args = (given["q"], given["k"], given["positions"], given["inverse_frequencies"], [], False,
            False, given["q_weight"], given["k_weight"], EPS)
    assert _C.rms_norm_rotary_if_supported(*args) is None
    assert _C.rotary_inputs_refusal(*args) == "all tensors must be HIP tensors"
    for function in (_C.rms_norm_rotary, _C.rms_norm_rotary_forward):
        with pytest.raises(RuntimeError, match="must be HIP tensors"):
            function(*args)
    with pytest.raises(RuntimeError, match="must be HIP tensors"):
        _C.rms_norm_rotary_backward(given["q"], given["k"], *args, 15)


# The C ABI.

FAKE = 1 << 20  # a non-null address; validation fails before it is touched
F32, F16, BF16, INT8 = range(4)


def heads(data=FAKE, outer=1 << 16, token=512, head=128):
    return _cabi.RlnHeads(data, outer, token, head)


def side(**changes):
    values = dict(heads=heads(), grad=heads(), count=4, weight=FAKE, weight_dtype=BF16,
                  output=FAKE, grad_weight=None)
    values.update(changes)
    return _cabi.RlnRotarySide(**values)


def table(**changes):
    values = dict(positions=FAKE, positions_type=0, axis_stride=64, outer_stride=8,
                  token_stride=1, frequencies=FAKE, wide_frequencies=0, axis_of_pair=None, axes=1,
                  pairs=64, interleaved=0)
    values.update(changes)
    return _cabi.RlnRotary(**values)


def run(backward=False, q=None, k=None, dtype=BF16, rotary=None, outer=2, inner=8, size=128,
        eps=EPS, workspace=None, workspace_bytes=0):
    """No argument set of these tests passes the checks."""
    q, k, rotary = q or side(), k or side(), rotary or table()
    library = _cabi.library()
    common = (ctypes.byref(q), ctypes.byref(k), dtype, ctypes.byref(rotary), outer, inner, size,
              eps)
    status = (library.rln_rotary_backward(*common, workspace, workspace_bytes, None) if backward
              else library.rln_rotary_forward(*common, None))
    assert status != 0
    return _cabi.last_error()


@pytest.mark.parametrize("backward", [False, True])
@pytest.mark.parametrize("changes,message", [
    (dict(dtype=INT8), "heads must use"),
    (dict(outer=0), "empty tensors"),
    (dict(inner=-1), "empty tensors"),
    (dict(inner=1 << 40), "number of tokens"),
    (dict(outer=1 << 20, inner=1 << 20), "number of tokens"),
    (dict(size=0), "head size: 0"),
    (dict(size=257), "head size: 257"),
    (dict(eps=-1.0), "eps"),
    (dict(rotary=table(positions=None)), "must not be null"),
    (dict(rotary=table(frequencies=None)), "must not be null"),
    (dict(rotary=table(pairs=65)), "pairs must be"),
    (dict(rotary=table(pairs=0)), "pairs must be"),
    (dict(rotary=table(axes=5)), "1 to 4 axes"),
    (dict(rotary=table(axes=0)), "1 to 4 axes"),
    (dict(rotary=table(positions_type=3)), "positions must use"),
    (dict(rotary=table(positions=FAKE + 4)), "positions is not aligned"),
    (dict(rotary=table(frequencies=FAKE + 4, wide_frequencies=1)), "frequencies is not aligned"),
    (dict(rotary=table(token_stride=1 << 61)), "positions: the strides overflow"),
    (dict(rotary=table(axis_of_pair=(ctypes.c_uint8 * 64)(*[0] * 63, 2), axes=2)), "past the last"),
    (dict(q=side(heads=heads(data=None))), "q must not be null"),
    (dict(q=side(heads=heads(data=FAKE + 1))), "q is not aligned"),
    (dict(k=side(heads=heads(outer=1 << 62))), "k: the strides overflow"),
    (dict(k=side(count=-1)), "number of heads"),
    (dict(k=side(count=1 << 17)), "number of heads"),
    (dict(q=side(count=0), k=side(count=0)), "empty tensors"),
    (dict(q=side(output=None)), "output must not be null"),
    (dict(q=side(output=FAKE + 1)), "output is not aligned"),
    (dict(q=side(weight_dtype=INT8)), "weight must use"),
    (dict(q=side(weight=FAKE + 1)), "weight is not aligned"),
    (dict(q=side(weight=None, grad_weight=FAKE)), "grad_weight without a weight"),
])
def test_refusals(backward, changes, message):
    assert message in run(backward, **changes)


@pytest.mark.parametrize("changes,message", [
    (dict(q=side(grad=heads(data=None))), "grad must not be null"),
    (dict(k=side(grad=heads(data=FAKE + 1))), "grad is not aligned"),
    (dict(q=side(grad_weight=FAKE)), "workspace too small"),
    (dict(k=side(grad_weight=FAKE), workspace=FAKE, workspace_bytes=64), "workspace too small"),
    (dict(k=side(grad_weight=FAKE + 1)), "grad_weight is not aligned"),
    (dict(q=side(grad_weight=FAKE), workspace=FAKE + 2, workspace_bytes=1 << 30),
     "workspace is not aligned"),
])
def test_backward_refusals(changes, message):
    assert message in run(True, **changes)


def test_a_forward_has_no_weight_gradient():
    assert "grad_weight without" in run(False, q=side(grad_weight=FAKE))


def test_workspace_sizes():
    size = _cabi.library().rln_rotary_backward_workspace_bytes
    for tokens in (1, 7, 100, 5000, (1 << 30) - 1):
        for q_heads, k_heads in ((1, 0), (4, 2), (64, 64), (1 << 16, 1)):
            for width in (1, 16, 72, 256):
                for dtype in (F32, F16, BF16):
                    for pairs in {1, width // 4, width // 2}:
                        got = size(1, tokens, q_heads, k_heads, width, pairs, dtype)
                        if pairs < 1 or 2 * pairs > width:
                            assert got == 0
                        else:
                            assert 4 * width <= got <= 2048 * 8 * width, (tokens, q_heads, width)
    for bad in ((0, 1, 1, 1, 16, 8, F32), (1, 1, 0, 0, 16, 8, F32), (1, 1, 1, 1, 257, 8, F32),
                (1, 1, 1, 1, 16, 9, F32), (1, 1, 1, 1, 16, 8, INT8), (1 << 30, 2, 1, 1, 16, 8, F32),
                (1, 1, 1 << 17, 1, 16, 8, F32)):
        assert size(*bad) == 0


def test_fake_shapes():
    from torch._subclasses.fake_tensor import FakeTensorMode

    ops = torch.ops.gfx1010_kernels
    with FakeTensorMode():
        q = torch.empty(2, 3, 4, 16, device="cuda", dtype=torch.bfloat16)
        k = torch.empty(2, 3, 2, 16, device="cuda", dtype=torch.bfloat16)
        positions = torch.empty(2, 3, device="cuda", dtype=torch.int64)
        frequencies, weight = torch.empty(8, device="cuda"), torch.empty(16, device="cuda")
        rest = (positions, frequencies, [], False, False, weight, None, EPS)
        for given in (k, None):
            q_out, k_out = ops.rotary_forward(q, given, *rest)
            assert q_out.shape == q.shape and q_out.dtype == q.dtype
            assert k_out.shape == (k.shape if given is not None else (0,))
            grads = ops.rotary_backward(q, given, q, None, *rest, 7)
            assert grads[0].shape == q.shape and grads[2].shape == weight.shape
            assert grads[1].shape == k_out.shape and grads[3].shape == (0,)


def fake_inputs(of_positions, of_frequencies):
    """Fake HIP tensors; either table may require a gradient."""
    q = torch.empty(2, 3, 4, 16, device="cuda").requires_grad_()
    positions = torch.empty(2, 3, device="cuda").requires_grad_(of_positions)
    return q, None, positions, torch.empty(8, device="cuda").requires_grad_(of_frequencies)


@pytest.mark.parametrize("of_positions,of_frequencies", [(True, False), (False, True)])
@pytest.mark.parametrize("heads_require", [True, False])
def test_the_registered_operator_drops_no_gradient(of_positions, of_frequencies, heads_require):
    """Its kernel runs without grad mode: what cannot be differentiated is refused above it."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    forward = torch.ops.gfx1010_kernels.rotary_forward
    rest = ([], False, False, None, None, EPS)
    with FakeTensorMode():
        given = fake_inputs(of_positions, of_frequencies)
        given[0].requires_grad_(heads_require)
        with pytest.raises(RuntimeError, match="positions and inverse_frequencies have no gradient"):
            forward(*given, *rest)
        with torch.no_grad():
            assert not forward(*given, *rest)[0].requires_grad
        assert forward(given[0].requires_grad_(), None, *(t.detach() for t in given[2:]),
                       *rest)[0].requires_grad


@pytest.mark.parametrize("of_positions,of_frequencies", [(True, False), (False, True)])
@pytest.mark.parametrize("implementation", ["gfx950", "gfx1010"])
@pytest.mark.parametrize("recorder", ["compile", "trace"])
def test_strict_modes_refuse_gradients_of_tables_in_graphs(of_positions, of_frequencies,
                                                           implementation, recorder, monkeypatch):
    from torch._subclasses.fake_tensor import FakeTensorMode

    if recorder == "compile":
        monkeypatch.setattr(torch.compiler, "is_compiling", lambda: True)
    else:
        monkeypatch.setattr(rotary, "graph_recorded", lambda: True)
    # What is reached behind the refusal: nothing of these calls.
    monkeypatch.setattr(rotary, "rms_norm_rotary_op", lambda *given: given)
    with FakeTensorMode():
        given = fake_inputs(of_positions, of_frequencies)
        with pytest.raises(RuntimeError, match="unavailable: positions and inverse_frequencies"):
            rms_norm_rotary(*given, implementation=implementation)
        with torch.no_grad():
            assert rms_norm_rotary(*given, implementation=implementation)[0] is given[0]


def sections_of_every_kind(numbers):
    import numpy as np

    return [tuple(numbers), list(numbers), torch.Size(numbers), np.array(numbers),
            torch.tensor(numbers), [np.int32(number) for number in numbers],
            tuple(float(number) for number in numbers)]


def test_sections_are_any_sequence_of_whole_numbers():
    given = dict(inputs(), implementation="torch")
    given["positions"] = torch.stack([given["positions"], given["positions"] + 3])
    expected = rms_norm_rotary(**given, sections=(5, 3))
    for sections in sections_of_every_kind((5, 3)):
        for a, b in zip(rms_norm_rotary(**given, sections=sections), expected):
            assert torch.equal(a, b), type(sections)
    for sections in ((5.5, 2.5), torch.tensor([5.5, 2.5]), (8.5, -0.5)):
        with pytest.raises(ValueError, match="whole numbers"):
            rms_norm_rotary(**given, sections=sections)


@pytest.mark.parametrize("backward", [False, True])
def test_limits_are_those_of_the_header(backward):
    """At each limit a later check answers, past it the limit's own."""
    last = side(output=None)
    for outer, inner in ((1, (1 << 30) - 1), ((1 << 30) - 1, 1), (3, (1 << 30) // 3)):
        assert "output must not" in run(backward, q=last, outer=outer, inner=inner)
    for outer, inner in ((1, 1 << 30), (1 << 30, 1), (1 << 15, 1 << 15), (3, (1 << 30) // 3 + 1)):
        assert "number of tokens" in run(backward, q=last, outer=outer, inner=inner)
    assert "output must not" in run(backward, q=side(output=None, count=1 << 16))
    assert "output must not" in run(backward, k=side(output=None, count=1 << 16))
    assert "number of heads" in run(backward, q=side(output=None, count=(1 << 16) + 1))
    assert "number of heads" in run(backward, k=side(output=None, count=(1 << 16) + 1))
    assert "output must not" in run(backward, q=last, size=256)
    assert "output must not" in run(backward, q=last, size=2, rotary=table(pairs=1))
    assert "pairs must be" in run(backward, q=last, size=1, rotary=table(pairs=1))
