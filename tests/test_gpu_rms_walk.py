"""The walking backward of the root-mean-square norm, which sums the weight's
gradient through a workspace: launches past the sizes that are summed in slab
blocks. Each test asserts that its launch is one, so that another threshold cannot
move it to the other form."""

import itertools

import pytest
import torch

import rms_reference as reference
from gfx1010_kernels import _cabi, residual_rms_norm

pytestmark = pytest.mark.gpu
EPS = 1e-6
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
CODE = {F32: 0, F16: 1, BF16: 2}
CHECKPOINTS = [None, torch.int8]
# Lengths by kernel: rows that share waves, one slot per lane, two, and (32-bit
# streams) four; on whole 32-bit words for every type, for 16-bit ones alone, for
# 32-bit ones alone; at both ends of a range.
LENGTHS = {
    F32: [1, 7, 64, 100, 128, 129, 200, 513, 516, 1001, 2046, 2048, 2049, 2052, 4095, 8192, 8193,
          8196, 8198, 16383, 16384],
    F16: [1, 9, 64, 130, 256, 257, 258, 260, 1027, 4094, 4096, 4097, 4098, 4100, 8193, 16383, 16384],
}
LENGTHS[BF16] = LENGTHS[F16]


def rows_past_slabs(hidden):
    """The least odd row count that is past both of the slab form's limits by a few."""
    return max(1, min(1027, (1 << 21) // hidden + 3)) | 1


def make(rows, hidden, x_dtype, branch_dtype, weight_dtype, grad_dtype, seed):
    generator = torch.Generator("cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, device="cuda", generator=generator)

    large = 1.0 + 15.0 * (normal(hidden) > 2.0)
    return ((normal(rows, hidden) * large).to(x_dtype),
            (0.5 * normal(rows, hidden)).to(branch_dtype),
            (1.0 + 0.1 * normal(hidden)).to(weight_dtype),
            [normal(rows, hidden).to(x_dtype), normal(rows, hidden).to(grad_dtype)])


def check(rows, hidden, x_dtype, branch_dtype, weight_dtype, grad_dtype, checkpoint):
    assert _cabi.rms_backward_workspace_bytes(rows, hidden, CODE[x_dtype]) > 0
    what = (rows, hidden, x_dtype, branch_dtype, weight_dtype, grad_dtype, checkpoint)
    x, branch, weight, upstream = make(rows, hidden, x_dtype, branch_dtype, weight_dtype,
                                       grad_dtype, hidden)
    leaves = [t.requires_grad_() for t in (x, branch, weight)]
    outputs = residual_rms_norm(*leaves, EPS, implementation="gfx950",
                                normalized_dtype=grad_dtype, checkpoint_dtype=checkpoint)
    grads = torch.autograd.grad(outputs, leaves, upstream, retain_graph=True)
    again = torch.autograd.grad(outputs, leaves, upstream)
    with torch.no_grad():
        u = reference.update(x, branch)
        kept = u if checkpoint is None else reference.checkpoint(u)[2]
        g, gw, size, terms = reference.gradients(u, kept, weight, EPS, *upstream)
        # Along the rows: those of one team (at least 256 teams), 8 of its wave, 8
        # teams, 8 partial sums of one lane and 64 lanes.
        depth = -(-rows // 256) + 8 + 8 + 8 + 64
        bounds = [reference.gradient_bound(g, size, x_dtype),
                  reference.gradient_bound(g, size, branch_dtype),
                  reference.weight_bound(gw, terms, depth, weight_dtype)]
        for grad, twin, value, bound, leaf, name in zip(
                grads, again, (g, g, gw), bounds, leaves, ("x", "branch", "weight")):
            assert grad.dtype == leaf.dtype and grad.shape == leaf.shape
            bits = torch.int32 if grad.element_size() == 4 else torch.int16
            assert torch.equal(grad.view(bits), twin.view(bits)), (what, name)
            bad = ~((grad.double() - value).abs() <= bound)
            assert not bad.any(), (what, name, int(bad.sum()), grad[bad][:4], value[bad][:4])


@pytest.mark.parametrize("checkpoint", CHECKPOINTS)
@pytest.mark.parametrize("weight_dtype,grad_dtype", list(itertools.product([F32, F16, BF16],
                                                                           repeat=2)))
@pytest.mark.parametrize("x_dtype,branch_dtype", list(itertools.product([F32, F16, BF16],
                                                                        repeat=2)))
def test_types(x_dtype, branch_dtype, weight_dtype, grad_dtype, checkpoint):
    for hidden in (120, 333, 520):
        check(1029, hidden, x_dtype, branch_dtype, weight_dtype, grad_dtype, checkpoint)


@pytest.mark.parametrize("checkpoint", CHECKPOINTS)
@pytest.mark.parametrize("grad_dtype", [F32, F16, BF16])
@pytest.mark.parametrize("x_dtype,hidden",
                         [(t, n) for t, lengths in LENGTHS.items() for n in lengths])
def test_lengths(x_dtype, hidden, grad_dtype, checkpoint):
    branch_dtype = {F32: BF16, F16: F32, BF16: F16}[grad_dtype]
    check(rows_past_slabs(hidden), hidden, x_dtype, branch_dtype, F32, grad_dtype, checkpoint)


@pytest.mark.parametrize("x_dtype", [F32, BF16])
@pytest.mark.parametrize("hidden,rows", [(3, 30011), (96, 16411), (384, 4099), (1000, 2055),
                                         (2050, 1539), (4096, 1025), (16384, 769)])
def test_teams_that_walk(x_dtype, hidden, rows):
    """More rows than teams: each walks over several, the last ones over one less."""
    for checkpoint in CHECKPOINTS:
        check(rows, hidden, x_dtype, BF16, F32, BF16, checkpoint)


# C ABI buffers.

def guarded(count, dtype):
    """`count` elements between two runs of a pattern, and their check."""
    size = torch.empty(0, dtype=dtype).element_size()
    whole = torch.full((4096 + count * size + 4096,), 0x5A, dtype=torch.uint8, device="cuda")
    inner = whole[4096:4096 + count * size].view(dtype)

    def check():
        assert (whole[:4096] == 0x5A).all() and (whole[4096 + count * size:] == 0x5A).all()
    return inner, check


@pytest.mark.parametrize("hidden", [1, 2, 4, 6, 63, 130, 514, 516, 520, 2055, 4096, 8195, 16382,
                                    16383])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_nothing_is_written_outside_the_outputs(hidden, dtype):
    rows, stream = rows_past_slabs(hidden), torch.cuda.current_stream().cuda_stream
    code = CODE[dtype]
    workspace_bytes = _cabi.rms_backward_workspace_bytes(rows, hidden, code)
    assert workspace_bytes > 0
    x, branch, weight, (grad_updated, grad_normalized) = make(rows, hidden, dtype, dtype, dtype,
                                                              dtype, 1)
    count, groups = rows * hidden, -(-hidden // 128)
    made = {name: guarded(*spec) for name, spec in dict(
        updated=(count, dtype), normalized=(count, dtype), rstd=(rows, F32),
        checkpoint=(count, torch.int8), checkpoint_scale=(rows * groups, F32)).items()}
    at = {name: inner.data_ptr() for name, (inner, _) in made.items()}
    _cabi.rms_forward(x.data_ptr(), code, weight.data_ptr(), code, at["normalized"], code, rows,
                      hidden, EPS, branch=branch.data_ptr(), branch_dtype=code,
                      updated=at["updated"], rstd=at["rstd"], checkpoint=at["checkpoint"],
                      checkpoint_scale=at["checkpoint_scale"], stream=stream)
    for kept, weighted in itertools.product(
            (dict(updated=at["updated"]),
             dict(checkpoint=at["checkpoint"], checkpoint_scale=at["checkpoint_scale"])),
            (True, False)):
        # NaN everywhere: what is not written shows.
        grads = {name: guarded(*spec) for name, spec in dict(
            grad_x=(count, dtype), grad_branch=(count, F16), grad_weight=(hidden, dtype)).items()}
        for inner, _ in grads.values():
            inner.fill_(float("nan"))
        workspace, workspace_check = guarded(workspace_bytes // 4, F32)
        workspace.fill_(float("nan"))
        _cabi.rms_backward(
            grad_updated.data_ptr(), grad_normalized.data_ptr(), code, code, weight.data_ptr(),
            code, at["rstd"], grads["grad_x"][0].data_ptr(), rows, hidden,
            grad_branch=grads["grad_branch"][0].data_ptr(), branch_dtype=CODE[F16],
            grad_weight=grads["grad_weight"][0].data_ptr() if weighted else None,
            workspace=workspace.data_ptr() if weighted else None,
            workspace_bytes=workspace_bytes if weighted else 0, stream=stream, **kept)
        for _, verify in [*made.values(), *grads.values()]:
            verify()
        workspace_check()
        assert grads["grad_x"][0].isfinite().all() and grads["grad_branch"][0].isfinite().all()
        assert grads["grad_weight"][0].isfinite().all() == weighted
        assert workspace.isfinite().all() == weighted
