"""The gated residual norm and the rotary norm of heads, as programs call them.

* ``call``: one ``gated_residual_rms_norm`` without a graph to record (prefill
  and decode steps of a served model, a denoising step of an image model).
* ``step``: the same and ``torch.autograd.grad`` of both outputs, the op's part
  of a training step.
* ``rotate``: one ``rms_norm_rotary`` of query and key heads without a graph.
* ``rotate_step``: the same and the gradients of the heads and their weights.

The definitions (``exact`` evaluates them in float64). Gated residual, per row
of H values, a the branch's norm (or the branch itself without a weight for it):

    a = branch / sqrt(mean(branch^2) + eps) * branch_weight
    u = residual_scale * x + branch_scale * gate * a, rounded to x's type
    r = 1 / sqrt(mean(u^2) + eps);  normalized = u * r * weight

``gate`` and ``weight`` hold one row for all, for each sample, or (the gate) for
each token. Rotary, per head of D values h:

    h = h / sqrt(mean(h^2) + eps) * head_weight (without a weight: h itself)
    pair i turns by positions[axis(i)] * inverse_frequencies[i]; the pairs are
    (i, i + P) of the first 2P values, or (2i, 2i + 1); the rest stays

``sections`` gives each axis (time, height, width) its number of pairs, in
blocks or taken in turns (axis 0 gets what the turns of the others leave).
A case names its tokens as ``batch`` x ``length``; ``strided`` takes the branch
as the first half of rows twice as wide, and the heads as parts of one joint
projection.
"""

from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

_PACKAGES = str(Path(__file__).resolve().parent.parent / "gfx1010-kernels_amd")
if _PACKAGES not in sys.path:
    sys.path.insert(0, _PACKAGES)

own = False

EPS = 1e-6
DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
SIZES = {"float32": 4, "float16": 2, "bfloat16": 2}


def _gated(name, kind, batch, length, hidden, x, branch, normalized, weight, *, post, gate,
           samples=False, residual_scale=1.0, branch_scale=1.0, strided=False):
    """``post``: the branch has a norm of its own; ``gate``: "none", "shared",
    "sample" or "token"; ``samples``: the last norm's weight is one per sample."""
    case = dict(kind=kind, batch=batch, length=length, hidden=hidden, x=x, branch=branch,
                normalized=normalized, weight=weight, post=post, gate=gate, samples=samples,
                residual_scale=residual_scale, branch_scale=branch_scale, strided=strided)
    return case if name is None else dict(case, name=name)


def _rotary(name, kind, batch, length, q_heads, k_heads, size, dtype, *, sections, norm,
            arrangement="blocks", interleaved=False, far=0, positions="int64", strided=False):
    """``sections``: pairs per axis, as "16,24,24"; ``far``: the first position."""
    case = dict(kind=kind, batch=batch, length=length, q_heads=q_heads, k_heads=k_heads,
                size=size, dtype=dtype, sections=sections, norm=norm, arrangement=arrangement,
                interleaved=interleaved, far=far, positions=positions, strided=strided)
    return case if name is None else dict(case, name=name)


def listed():
    bf16, fp16, fp32 = "bfloat16", "float16", "float32"
    return [
        # A decode step of 8 sequences, norms before and after the block: latency.
        _gated("decode", "call", 8, 1, 4096, bf16, bf16, bf16, bf16, post=True, gate="none"),
        # Prefill of one ragged prompt, a scaled residual; the branch is a part of wider rows.
        _gated("prefill_ragged", "call", 1, 6001, 2880, bf16, bf16, bf16, bf16, post=True,
               gate="none", branch_scale=0.22, strided=True),
        # A denoising step of two images whose gate and weight depend on the sample.
        _gated("image_gated", "call", 2, 4429, 2304, bf16, bf16, bf16, bf16, post=True,
               gate="sample", samples=True),
        # GPT-2-small-shaped training batch with a learned scale of the branch.
        _gated("train_768", "step", 8, 1024, 768, fp32, bf16, bf16, fp32, post=False,
               gate="shared"),
        # All in 32 bits, rows of an odd length, a gate for each token.
        _gated("train_odd", "step", 3, 1237, 1001, fp32, fp32, fp32, fp32, post=True,
               gate="token", residual_scale=1.25),
        # A large batch all in bf16, gate and weight by sample.
        _gated("train_large", "step", 16, 1024, 4096, bf16, bf16, bf16, bf16, post=True,
               gate="sample", samples=True),
        # A decode step of 16 sequences at far positions, heads normed, grouped keys: latency.
        _rotary("decode_heads", "rotate", 16, 1, 32, 8, 128, bf16, sections="64", norm=True,
                far=131071),
        # Prefill of a video prompt, three axes, heads as parts of a joint projection.
        _rotary("prefill_video", "rotate", 1, 6001, 28, 4, 128, bf16, sections="16,24,24",
                norm=False, strided=True),
        # Images of two axes, neighbouring pairs, heads of 72 values.
        _rotary("image_pairs", "rotate", 2, 4429, 16, 16, 72, fp16, sections="18,18", norm=True,
                interleaved=True, positions="float32"),
        # Part of a 32-bit head turned, no norm, far positions, an odd batch.
        _rotary("train_partial", "rotate_step", 3, 1237, 15, 5, 80, fp32, sections="16",
                norm=False, far=1000003),
        # GPT-2-small-shaped training batch with normed heads.
        _rotary("train_heads", "rotate_step", 8, 1024, 12, 12, 64, fp16, sections="32", norm=True,
                strided=True),
        # A large training batch, axes in turns, grouped keys.
        _rotary("train_grouped", "rotate_step", 4, 4096, 32, 8, 128, bf16, sections="24,20,20",
                norm=True, arrangement="cyclic"),
    ]


def _log_uniform(rng, low, high):
    return math.exp(rng.uniform(math.log(low), math.log(high)))


def _draw_gated(rng):
    kind = rng.choice(["call", "step"])
    hidden = round(_log_uniform(rng, 64, 16384))
    hidden = hidden | 1 if rng.random() < 1 / 3 else max(64, hidden // 8 * 8)
    low = hidden if kind == "call" else max(hidden, 1 << 16)
    high = 1 << (25 if kind == "call" else 24)
    rows = max(1, round(_log_uniform(rng, low, max(high, 2 * hidden)) / hidden))
    batch = min(rows, rng.choice([1, 2, 3, 8, 16]))
    half = rng.choice(["float16", "bfloat16"])
    x = rng.choice([half, "float32"])
    return _gated(None, kind, batch, max(1, rows // batch), hidden, x, rng.choice([x, half]),
                  rng.choice([x, half]), rng.choice([x, "float32"]), post=rng.random() < 0.7,
                  gate=rng.choice(["none", "shared", "sample", "token"]),
                  samples=rng.random() < 0.3,
                  residual_scale=rng.choice([1.0, 1.0, round(rng.uniform(0.5, 2.0), 3)]),
                  branch_scale=rng.choice([1.0, round(rng.uniform(0.1, 1.0), 3)]),
                  strided=rng.random() < 0.2)


def _draw_rotary(rng):
    kind = rng.choice(["rotate", "rotate_step"])
    size = rng.choice([32, 48, 64, 72, 80, 96, 100, 128, 128, 160, 192, 256, rng.randrange(16, 257)])
    k_heads = rng.choice([1, 2, 3, 4, 8, 12, 16])
    q_heads = k_heads * rng.choice([1, 1, 2, 3, 4, 5, 7, 8])
    width = (q_heads + k_heads) * size
    low = width if kind == "rotate" else max(width, 1 << 16)
    tokens = max(1, round(_log_uniform(rng, low, 1 << 25) / width))
    batch = min(tokens, rng.choice([1, 1, 2, 3, 8]))
    pairs = max(4, size // 2 if rng.random() < 0.7 else size // rng.choice([4, 5, 8]))
    axes = rng.choice([1, 1, 2, 3, 4])
    sections = [pairs // axes] * axes
    sections[0] += pairs - sum(sections)
    return _rotary(None, kind, batch, max(1, tokens // batch), q_heads, k_heads, size,
                   rng.choice(["float16", "bfloat16", "bfloat16", "float32"]),
                   sections=",".join(map(str, sections)), norm=rng.random() < 0.6,
                   arrangement=rng.choice(["blocks", "cyclic"]),
                   interleaved=rng.random() < 0.4,
                   far=rng.choice([0, 0, round(_log_uniform(rng, 1, 1 << 20))]),
                   positions=rng.choice(["int64", "int32", "float32"]),
                   strided=rng.random() < 0.4)


def draw(rng):
    """One more case: either operator in either direction. Gated rows of 64 to
    16384 values (every third length odd), from one token to 2^25 elements (2^24 in
    a step); heads of 16 to 256 values, 1 to 4 axes, from one token to 2^25."""
    return _draw_gated(rng) if rng.random() < 0.5 else _draw_rotary(rng)


# Inputs, from the seed alone.

def _normal(generator):
    def normal(size, dtype, scale=1.0, mean=0.0):
        values = torch.randn(size, device="cuda", generator=generator)
        return values.mul_(scale).add_(mean).to(DTYPES[dtype])
    return normal


def _gated_inputs(case, seed):
    """A residual stream some of whose columns are far larger than the rest, as
    trained models have them, a branch beside it, weights around one, gates
    around zero, upstream gradients."""
    generator = torch.Generator("cuda").manual_seed(seed)
    normal = _normal(generator)
    batch, length, hidden = case["batch"], case["length"], case["hidden"]
    shape = (batch, length, hidden)
    large = torch.rand(hidden, device="cuda", generator=generator) < 0.004
    inputs = dict(x=(normal(shape, "float32") * (1.0 + 15.0 * large)).to(DTYPES[case["x"]]))
    width = 2 * hidden if case["strided"] else hidden
    inputs["branch"] = normal((batch, length, width), case["branch"], 0.5)[..., :hidden]
    inputs["weight"] = normal((batch, 1, hidden) if case["samples"] else (hidden,),
                              case["weight"], 0.1, 1.0)
    inputs["branch_weight"] = normal(hidden, case["weight"], 0.1, 1.0) if case["post"] else None
    gate = {"none": None, "shared": (hidden,), "sample": (batch, 1, hidden),
            "token": shape}[case["gate"]]
    inputs["gate"] = None if gate is None else normal(gate, case["x"], 0.5)
    if case["kind"] == "step":
        inputs["grad_updated"] = normal(shape, case["x"], 0.1)
        inputs["grad_normalized"] = normal(shape, case["normalized"], 0.1)
    return inputs


def _sections(case):
    return tuple(int(part) for part in case["sections"].split(","))


def _positions(case, generator):
    """[axes, batch, length]: time counts on from ``far``; height and width walk a
    grid, so that neighbouring tokens share some of their positions."""
    batch, length = case["batch"], case["length"]
    index = torch.arange(length, device="cuda")
    first = torch.randint(0, 64, (batch, 1), device="cuda", generator=generator) + case["far"]
    side = max(1, math.isqrt(length))
    axes = [first + index, (first + index // side).expand(batch, length),
            (first + index % side).expand(batch, length), (first + index // 2)]
    positions = torch.stack(axes[:len(_sections(case))])
    if case["positions"] == "float32":  # between the whole ones, as resized grids have them
        return positions.float() * 0.75
    return positions.to(torch.int32 if case["positions"] == "int32" else torch.int64)


def _rotary_inputs(case, seed):
    generator = torch.Generator("cuda").manual_seed(seed)
    normal = _normal(generator)
    tokens, size = (case["batch"], case["length"]), case["size"]
    q_heads, k_heads, dtype = case["q_heads"], case["k_heads"], case["dtype"]
    if case["strided"]:
        joint = normal((*tokens, (q_heads + 2 * k_heads) * size), dtype)
        q, k, _ = joint.split([q_heads * size, k_heads * size, k_heads * size], -1)
        q, k = q.unflatten(-1, (q_heads, size)), k.unflatten(-1, (k_heads, size))
    else:
        q, k = normal((*tokens, q_heads, size), dtype), normal((*tokens, k_heads, size), dtype)
    pairs = sum(_sections(case))
    ladder = torch.arange(pairs, dtype=torch.float64, device="cuda") / pairs
    inputs = dict(q=q, k=k, positions=_positions(case, generator),
                  frequencies=(10000.0 ** -ladder).float(), q_weight=None, k_weight=None)
    if case["norm"]:
        inputs["q_weight"] = normal(size, dtype, 0.1, 1.0)
        inputs["k_weight"] = normal(size, dtype, 0.1, 1.0)
    if case["kind"] == "rotate_step":
        inputs["grad_q"] = normal(q.shape, dtype, 0.1)
        inputs["grad_k"] = normal(k.shape, dtype, 0.1)
    return inputs


_GATED_LEAVES = ("x", "branch", "weight", "branch_weight", "gate")
_ROTARY_LEAVES = ("q", "k", "q_weight", "k_weight")


def prepare(case, seed):
    rotary = case["kind"].startswith("rotate")
    state = _rotary_inputs(case, seed) if rotary else _gated_inputs(case, seed)
    if case["kind"].endswith("step"):
        leaves = []
        for name in _ROTARY_LEAVES if rotary else _GATED_LEAVES:
            if state[name] is not None:
                state[name] = state[name].detach().requires_grad_()
                leaves.append(state[name])
        state["leaves"] = leaves
    state["kind"] = case["kind"]
    if rotary:
        state.update(sections=_sections(case), arrangement=case["arrangement"],
                     interleaved=case["interleaved"])
    else:
        state.update(dtype=DTYPES[case["normalized"]], residual_scale=case["residual_scale"],
                     branch_scale=case["branch_scale"])
    return state


# The plain forms.

def _wide(tensor):
    return None if tensor is None else tensor.float()


def _rstd(values):
    return 1.0 / torch.sqrt(values.square().mean(-1, keepdim=True) + EPS)


def _plain_gated(state):
    """(updated, normalized) and what the gradients need."""
    unit = state["branch"].float()
    scale = torch.ones_like(unit[..., :1])
    if state["branch_weight"] is not None:
        scale = _rstd(unit)
        unit = unit * scale
    factor = torch.full_like(unit[0, 0], state["branch_scale"])
    if state["branch_weight"] is not None:
        factor = factor * state["branch_weight"].float()
    if state["gate"] is not None:
        factor = factor * state["gate"].float()
    updated = (state["residual_scale"] * state["x"].float() + factor * unit).to(state["x"].dtype)
    values = updated.float()
    rstd = _rstd(values)
    normalized = (values * rstd * state["weight"].float()).to(state["dtype"])
    return updated, normalized, unit, scale, factor, values * rstd, rstd


def _summed(values, like):
    """Summed over the dimensions that ``like`` repeats over, in 64 bits: long sums."""
    over = [0, 1] if like.ndim == 1 else [d for d in (0, 1) if like.shape[d] == 1]
    if over:
        values = values.sum(over, keepdim=True, dtype=torch.float64)
    return values.reshape(like.shape).to(like.dtype)


def _plain_step(state):
    updated, normalized, unit, scale, factor, normed, rstd = _plain_gated(state)
    upstream = state["grad_normalized"].float()
    product = upstream * state["weight"].float()
    gradient = state["grad_updated"].float() + rstd * (
        product - normed * (product * normed).mean(-1, keepdim=True))
    inner = gradient * factor
    if state["branch_weight"] is not None:
        inner = scale * (inner - unit * (inner * unit).mean(-1, keepdim=True))
    answer = [updated, normalized, (state["residual_scale"] * gradient).to(updated.dtype),
              inner.to(state["branch"].dtype), _summed(upstream * normed, state["weight"])]
    each = state["branch_scale"] * gradient * unit
    weight, gate = _wide(state["branch_weight"]), _wide(state["gate"])
    if weight is not None:
        answer.append(_summed(each if gate is None else each * gate, state["branch_weight"]))
    if gate is not None:
        answer.append(_summed(each if weight is None else each * weight, state["gate"]))
    return tuple(answer)


def _axis_of_pairs(sections, arrangement):
    """The axis of each pair."""
    if arrangement == "blocks":
        return [axis for axis, count in enumerate(sections) for _ in range(count)]
    taken = [0] * sum(sections)
    for axis in range(1, len(sections)):
        for turn in range(sections[axis]):
            place = axis + turn * len(sections)
            if place < len(taken):
                taken[place] = axis
    return taken


def _plain_angles(state):
    """cos and sin [batch, length, 1, pairs] in 32 bits, of angles in 64."""
    axes = torch.tensor(_axis_of_pairs(state["sections"], state["arrangement"]), device="cuda")
    angles = state["positions"].double()[axes].movedim(0, -1) * state["frequencies"].double()
    return angles.cos().float().unsqueeze(-2), angles.sin().float().unsqueeze(-2)


def _pairs_of(values, pairs, interleaved):
    turned = values[..., :2 * pairs]
    if interleaved:
        return turned[..., 0::2], turned[..., 1::2]
    return turned[..., :pairs], turned[..., pairs:]


def _turned(values, cos, sin, interleaved):
    pairs = cos.shape[-1]
    first, second = _pairs_of(values, pairs, interleaved)
    first, second = first * cos - second * sin, first * sin + second * cos
    if interleaved:
        turned = torch.stack([first, second], -1).flatten(-2)
    else:
        turned = torch.cat([first, second], -1)
    return torch.cat([turned, values[..., 2 * pairs:]], -1)


def _plain_rotate(state):
    cos, sin = _plain_angles(state)
    answer = []
    for name in ("q", "k"):
        values, weight = state[name].float(), state[name + "_weight"]
        if weight is not None:
            values = values * _rstd(values) * weight.float()
        answer.append(_turned(values, cos, sin, state["interleaved"]).to(state[name].dtype))
    return tuple(answer)


def _plain_rotate_step(state):
    cos, sin = _plain_angles(state)
    gradients, sums = [], []
    for name in ("q", "k"):
        heads, weight = state[name], state[name + "_weight"]
        gradient = _turned(state["grad_" + name].float(), cos, -sin, state["interleaved"])
        if weight is not None:
            values = heads.float()
            rstd = _rstd(values)
            unit, product = values * rstd, gradient * weight.float()
            sums.append((gradient * unit).sum((0, 1, 2), dtype=torch.float64).to(weight.dtype))
            gradient = rstd * (product - unit * (product * unit).mean(-1, keepdim=True))
        gradients.append(gradient.to(heads.dtype))
    return (*_plain_rotate(state), *gradients, *sums)


# The framework's calls.

def _own_gated(state):
    from gfx1010_kernels import gated_residual_rms_norm

    return gated_residual_rms_norm(
        state["x"], state["branch"], state["weight"], EPS, branch_weight=state["branch_weight"],
        gate=state["gate"], residual_scale=state["residual_scale"],
        branch_scale=state["branch_scale"], normalized_dtype=state["dtype"])


def _own_rotate(state):
    from gfx1010_kernels import rms_norm_rotary

    return rms_norm_rotary(
        state["q"], state["k"], state["positions"], state["frequencies"],
        sections=state["sections"], arrangement=state["arrangement"],
        interleaved=state["interleaved"], q_weight=state["q_weight"], k_weight=state["k_weight"],
        eps=EPS)


def run(state):
    kind = state["kind"]
    if own and kind.endswith("step"):
        outputs = _own_gated(state) if kind == "step" else _own_rotate(state)
        upstream = (("grad_updated", "grad_normalized") if kind == "step"
                    else ("grad_q", "grad_k"))
        return (*outputs, *torch.autograd.grad(outputs, state["leaves"],
                                               [state[name] for name in upstream]))
    with torch.no_grad():
        if kind == "step":
            return _plain_step(state)
        if kind == "rotate_step":
            return _plain_rotate_step(state)
        if kind == "rotate":
            return _own_rotate(state) if own else _plain_rotate(state)
        return _own_gated(state) if own else _plain_gated(state)[:2]


def work(case):
    """Compulsory traffic: every input read once and every output written once,
    what a training forward keeps for its backward read once more."""
    if case["kind"].startswith("rotate"):
        tokens, size = case["batch"] * case["length"], SIZES[case["dtype"]]
        count = tokens * (case["q_heads"] + case["k_heads"]) * case["size"]
        small = len(_sections(case)) * tokens * (8 if case["positions"] == "int64" else 4)
        total, flops = 2 * size * count + small, (6.0 + 4.0 * case["norm"]) * count
        if case["kind"] == "rotate_step":
            total += (3 if case["norm"] else 2) * size * count + small
            flops += (6.0 + 10.0 * case["norm"]) * count
        return {"bytes": total, "flops": flops}
    hidden, rows = case["hidden"], case["batch"] * case["length"]
    count = rows * hidden
    x, branch, normalized = SIZES[case["x"]], SIZES[case["branch"]], SIZES[case["normalized"]]
    weights = hidden * SIZES[case["weight"]] * ((case["batch"] if case["samples"] else 1)
                                                + case["post"])
    gate = x * hidden * {"none": 0, "shared": 1, "sample": case["batch"],
                         "token": rows}[case["gate"]]
    total = count * (x + branch + x + normalized) + weights + gate
    flops = 14.0 * count
    if case["kind"] == "step":
        # updated, branch, gate and both upstream gradients -> every gradient
        total += count * (x + branch + x + normalized) + weights + gate
        total += count * (x + branch) + weights + gate
        flops += 30.0 * count
    return {"bytes": total, "flops": flops}


# The definitions in 64 bits.

def _exact_gated(case, seed):
    inputs = _gated_inputs(case, seed)
    batch, length, hidden = case["batch"], case["length"], case["hidden"]
    step = case["kind"] == "step"

    def row(name, sample, a, b):
        """A weight's or gate's rows for tokens a to b of one sample."""
        tensor = inputs[name]
        if tensor is None:
            return 1.0
        if tensor.ndim == 1:
            return tensor.double()
        return (tensor[sample, a:b] if tensor.shape[1] == length else tensor[sample]).double()

    pieces = {name: [] for name in ("u", "y", "gx", "gb", "gate")}
    shape = (batch, hidden)
    sums = {name: torch.zeros(shape, dtype=torch.float64, device="cuda")
            for name in ("weight", "branch_weight", "gate")}
    tokens = max(1, (1 << 22) // hidden)
    for sample in range(batch):
        for a in range(0, length, tokens):
            b = min(length, a + tokens)
            x, branch = (inputs[name][sample, a:b].double() for name in ("x", "branch"))
            inner = 1.0
            if case["post"]:
                inner = (branch.square().mean(-1, keepdim=True) + EPS).rsqrt()
            bw, gate = row("branch_weight", sample, a, b), row("gate", sample, a, b)
            weight = row("weight", sample, a, b)
            unit = branch * inner
            u = (case["residual_scale"] * x + case["branch_scale"] * gate * bw * unit)
            u = u.to(inputs["x"].dtype).double()
            r = (u.square().mean(-1, keepdim=True) + EPS).rsqrt()
            pieces["u"].append(u)
            pieces["y"].append(u * r * weight)
            if not step:
                continue
            gu, gy = (inputs[name][sample, a:b].double()
                      for name in ("grad_updated", "grad_normalized"))
            p = gy * weight
            g = gu + r * p - u * r ** 3 * (p * u).mean(-1, keepdim=True)
            pieces["gx"].append(case["residual_scale"] * g)
            q = case["branch_scale"] * g
            z = q * gate * bw
            if case["post"]:
                pieces["gb"].append(inner * z
                                    - branch * inner ** 3 * (z * branch).mean(-1, keepdim=True))
            else:
                pieces["gb"].append(z)
            sums["weight"][sample] += (gy * u * r).sum(0)
            sums["branch_weight"][sample] += (q * gate * unit).sum(0)
            if case["gate"] == "token":
                pieces["gate"].append(q * bw * unit)
            else:
                sums["gate"][sample] += (q * bw * unit).sum(0)

    def whole(name):
        return torch.cat(pieces[name]).view(batch, length, hidden)

    def summed(name, each):
        return sums[name].unsqueeze(1) if each else sums[name].sum(0)

    answer = [whole("u"), whole("y")]
    if step:
        answer += [whole("gx"), whole("gb"), summed("weight", case["samples"])]
        if case["post"]:
            answer.append(summed("branch_weight", False))
        if case["gate"] == "token":
            answer.append(whole("gate"))
        elif case["gate"] != "none":
            answer.append(summed("gate", case["gate"] == "sample"))
    return tuple(answer)


def _exact_rotary(case, seed):
    """Pairs as complex numbers, turned by a product with exp(i angle)."""
    inputs = _rotary_inputs(case, seed)
    batch, length, size = case["batch"], case["length"], case["size"]
    sections = _sections(case)
    pairs, interleaved = sum(sections), case["interleaved"]
    axes = _axis_of_pairs(sections, case["arrangement"])

    def turn(values, a, b, sample, back):
        where = inputs["positions"][:, sample, a:b].double()
        angles = torch.stack([where[axis] for axis in axes], -1) * inputs["frequencies"].double()
        factor = torch.polar(torch.ones_like(angles), -angles if back else angles).unsqueeze(1)
        if interleaved:
            real, imaginary = values[..., 0:2 * pairs:2], values[..., 1:2 * pairs:2]
        else:
            real, imaginary = values[..., :pairs], values[..., pairs:2 * pairs]
        product = torch.complex(real, imaginary) * factor
        turned = values.clone()
        if interleaved:
            turned[..., 0:2 * pairs:2], turned[..., 1:2 * pairs:2] = product.real, product.imag
        else:
            turned[..., :pairs], turned[..., pairs:2 * pairs] = product.real, product.imag
        return turned

    outputs, gradients, sums = [], [], []
    for name in ("q", "k"):
        heads, weight = inputs[name], inputs[name + "_weight"]
        forward, backward = [], []
        total = torch.zeros(size, dtype=torch.float64, device="cuda")
        tokens = max(1, (1 << 22) // (heads.shape[2] * size))
        for sample in range(batch):
            for a in range(0, length, tokens):
                b = min(length, a + tokens)
                values = heads[sample, a:b].double()
                r = (values.square().mean(-1, keepdim=True) + EPS).rsqrt()
                normed = values if weight is None else values * r * weight.double()
                forward.append(turn(normed, a, b, sample, False))
                if case["kind"] == "rotate":
                    continue
                g = turn(inputs["grad_" + name][sample, a:b].double(), a, b, sample, True)
                if weight is not None:
                    total += (g * values * r).sum((0, 1))
                    p = g * weight.double()
                    g = r * p - values * r ** 3 * (p * values).mean(-1, keepdim=True)
                backward.append(g)
        outputs.append(torch.cat(forward).view(heads.shape))
        if case["kind"] == "rotate_step":
            gradients.append(torch.cat(backward).view(heads.shape))
            if weight is not None:
                sums.append(total)
    return (*outputs, *gradients, *sums)


def exact(case, seed):
    return (_exact_rotary if case["kind"].startswith("rotate") else _exact_gated)(case, seed)
