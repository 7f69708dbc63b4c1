"""The root-mean-square norm operators, as programs call them.

* ``call``: one ``residual_rms_norm`` without a graph to record (prefill and
  decode steps of a served model).
* ``step``: ``residual_rms_norm`` and ``torch.autograd.grad`` of both outputs,
  the op's part of a training step; ``checkpoint`` keeps the norm's input for
  the backward in 8 bits.
* ``quant``: ``residual_rms_norm_quantized`` of a served model with 8-bit
  products; e4m3 comes back as it is, int8 widened by ``dequantize`` for a
  consumer in bf16.

The definition, per row of H values (``exact`` evaluates it in float64):

    u = x + branch, rounded to x's type;  r = 1 / sqrt(mean(u^2) + eps)
    normalized = u * r * weight
    backward: p = gy * weight;  g = gu + r * (p - u * r * mean(p * u * r)),
              the gradient of x and of branch;  sum of gy * u * r over the
              rows, that of weight
    8 bits: v = u * weight (fp32);  a = max |v| of a group of columns;
            q = round(v * (Q / a)), Q = 127 or 448;  scale = a / Q * r
    checkpoint: a = max |u| of 128 columns; the backward takes
            round(u * (127 / a)) * (a / 127) for u

A case names its rows as ``batch`` x ``length``; ``strided`` takes the branch
as the first half of rows twice as wide (one part of a joint projection).
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
DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16,
          "int8": torch.int8, "e4m3": torch.float8_e4m3fn}
SIZES = {"float32": 4, "float16": 2, "bfloat16": 2, "int8": 1, "e4m3": 1}
TOP = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}
CHECKPOINT_GROUP = 128
TINY = 2.0 ** -100  # the least maximum of a group


def _case(name, kind, batch, length, hidden, x, branch, normalized, weight, *, group=0,
          checkpoint=False, strided=False):
    case = dict(kind=kind, batch=batch, length=length, hidden=hidden, x=x, branch=branch,
                normalized=normalized, weight=weight, group=group, checkpoint=checkpoint,
                strided=strided)
    return case if name is None else dict(case, name=name)


def listed():
    bf16, fp16, fp32 = "bfloat16", "float16", "float32"
    return [
        # A decode step of 8 sequences, all in bf16: one call, bound by latency.
        _case("decode", "call", 8, 1, 4096, bf16, bf16, bf16, bf16),
        # Prefill of one ragged prompt; the branch is a part of wider rows.
        _case("prefill_ragged", "call", 1, 6001, 2880, bf16, bf16, bf16, bf16, strided=True),
        # A decode step of 64 sequences in front of an e4m3 product, a scale a token.
        _case("decode_e4m3", "quant", 64, 1, 5120, bf16, bf16, "e4m3", bf16),
        # Prefill of 8 prompts in front of a product with scales by blocks of 128.
        _case("prefill_e4m3_groups", "quant", 8, 1024, 4096, bf16, bf16, "e4m3", bf16, group=128),
        # int8 activations of odd batches, a scale a token, widened again.
        _case("prefill_int8", "quant", 3, 1367, 1600, fp16, fp16, "int8", fp16),
        # A large evaluation batch on a 32-bit stream, int8 in groups of 64.
        _case("eval_int8_groups", "quant", 32, 1024, 2048, fp32, bf16, "int8", fp32, group=64),
        # GPT-2-small-shaped training batch, 32-bit stream, bf16 sublayers.
        _case("train_768", "step", 8, 1024, 768, fp32, bf16, bf16, fp32),
        # All in 32 bits, rows of an odd length.
        _case("train_odd", "step", 3, 1237, 1001, fp32, fp32, fp32, fp32),
        # A large batch all in bf16.
        _case("train_large", "step", 16, 1024, 4096, bf16, bf16, bf16, bf16),
        # The character-level GPT's microstep with 8-bit checkpoints.
        _case("char_gpt_checkpoint", "step", 1, 1024, 384, fp32, fp16, fp16, fp32,
              checkpoint=True),
        # A middle-sized batch all in bf16 with 8-bit checkpoints.
        _case("train_checkpoint", "step", 8, 2048, 2048, bf16, bf16, bf16, bf16, checkpoint=True),
        # The largest: long rows of a 32-bit stream, 8-bit checkpoints.
        _case("train_checkpoint_large", "step", 8, 1024, 8192, fp32, bf16, bf16, fp32,
              checkpoint=True),
    ]


def _log_uniform(rng, low, high):
    return math.exp(rng.uniform(math.log(low), math.log(high)))


def draw(rng):
    """One more case: any kind and types, a row length from 64 to 16384 (every
    third one odd), from one token to 2^25 elements."""
    kind = rng.choice(["call", "step", "step", "quant", "quant"])
    hidden = round(_log_uniform(rng, 64, 16384))
    hidden = hidden | 1 if rng.random() < 1 / 3 else max(64, hidden // 8 * 8)
    low, high = {"call": (hidden, 1 << 25), "quant": (hidden, 1 << 25),
                 "step": (1 << 16, 1 << 25)}[kind]
    rows = max(1, round(_log_uniform(rng, max(low, hidden), max(high, 2 * hidden)) / hidden))
    batch = min(rows, rng.choice([1, 1, 2, 3, 8]))
    half = rng.choice(["float16", "bfloat16"])
    x = rng.choice([half, "float32"])
    branch = rng.choice([x, half])
    normalized = rng.choice(["e4m3", "int8"]) if kind == "quant" else rng.choice([x, half])
    return _case(None, kind, batch, max(1, rows // batch), hidden, x, branch, normalized,
                 rng.choice([x, "float32"]),
                 group=rng.choice([0, 0, 32, 64, 128, 256]) if kind == "quant" else 0,
                 checkpoint=kind == "step" and rng.random() < 0.5,
                 strided=rng.random() < 0.2)


def _inputs(case, seed):
    """Inputs from the seed alone: a residual stream some of whose columns are
    far larger than the rest, as trained models have them, a branch beside it,
    a weight around one, upstream gradients."""
    generator = torch.Generator("cuda").manual_seed(seed)
    hidden = case["hidden"]
    shape = (case["batch"], case["length"], hidden)

    def normal(size, scale=1.0, mean=0.0):
        values = torch.randn(size, device="cuda", generator=generator)
        return values.mul_(scale).add_(mean)

    large = torch.rand(hidden, device="cuda", generator=generator) < 0.004
    inputs = dict(x=normal(shape).mul_(1.0 + 15.0 * large).to(DTYPES[case["x"]]),
                  weight=normal(hidden, 0.1, 1.0).to(DTYPES[case["weight"]]))
    width = 2 * hidden if case["strided"] else hidden
    inputs["branch"] = normal((*shape[:2], width), 0.5).to(DTYPES[case["branch"]])[..., :hidden]
    if case["kind"] == "step":
        inputs["grad_updated"] = normal(shape, 0.1).to(DTYPES[case["x"]])
        inputs["grad_normalized"] = normal(shape, 0.1).to(DTYPES[case["normalized"]])
    return inputs


def prepare(case, seed):
    state = _inputs(case, seed)
    if case["kind"] == "step":
        state["branch"] = state["branch"].detach()
        for name in ("x", "branch", "weight"):
            state[name].requires_grad_()
    state.update(kind=case["kind"], dtype=DTYPES[case["normalized"]], group=case["group"] or None,
                 checkpoint=torch.int8 if case["checkpoint"] else None)
    return state


# The plain forms.

def _group_maximum(values, group):
    """The largest magnitude of each group of columns, the last one shorter."""
    missing = -values.shape[-1] % group
    padded = torch.cat([values, values.new_zeros(*values.shape[:-1], missing)], -1)
    return padded.view(*values.shape[:-1], -1, group).abs().amax(-1).clamp(min=TINY)


def _spread(groups, group, hidden):
    """Each group's value at each of its columns."""
    return groups.repeat_interleave(group, -1)[..., :hidden]


def _plain_forward(state):
    updated = (state["x"].float() + state["branch"].float()).to(state["x"].dtype)
    values = updated.float()
    rstd = 1.0 / torch.sqrt(values.square().mean(-1, keepdim=True) + EPS)
    return updated, values, rstd


def _plain_call(state):
    updated, values, rstd = _plain_forward(state)
    return updated, (values * rstd * state["weight"].float()).to(state["dtype"])


def _plain_quantized(state):
    updated, values, rstd = _plain_forward(state)
    hidden, top = values.shape[-1], TOP[state["dtype"]]
    group = state["group"] or hidden
    values = values * state["weight"].float()
    largest = _group_maximum(values, group)
    steps = values * _spread(torch.full_like(largest, top) / largest, group, hidden)
    scale = largest / torch.full_like(largest, top) * rstd
    if state["dtype"] == torch.int8:
        whole = steps.round().clamp(-top, top)
        return updated, (whole * _spread(scale, group, hidden)).to(torch.bfloat16), scale
    return updated, steps.clamp(-top, top).to(state["dtype"]), scale


def _plain_step(state):
    updated, values, rstd = _plain_forward(state)
    weight = state["weight"].float()
    normalized = (values * rstd * weight).to(state["dtype"])
    if state["checkpoint"] is not None:
        hidden, group = values.shape[-1], CHECKPOINT_GROUP
        largest = _group_maximum(values, group)
        top = torch.full_like(largest, 127.0)
        kept = (values * _spread(top / largest, group, hidden)).round()
        values = kept * _spread(largest / top, group, hidden)
    upstream = state["grad_normalized"].float()
    unit = values * rstd
    product = upstream * weight
    shared = (product * unit).mean(-1, keepdim=True)
    gradient = state["grad_updated"].float() + rstd * (product - unit * shared)
    # Sums over the rows in 64 bits: long ones.
    grad_weight = (upstream * unit).sum((0, 1), dtype=torch.float64)
    return (updated, normalized, gradient.to(updated.dtype), gradient.to(state["branch"].dtype),
            grad_weight.to(state["weight"].dtype))


# The framework's calls.

def _own_call(state):
    from gfx1010_kernels import residual_rms_norm

    return residual_rms_norm(state["x"], state["branch"], state["weight"], EPS,
                             normalized_dtype=state["dtype"])


def _own_quantized(state):
    from gfx1010_kernels import dequantize, residual_rms_norm_quantized

    updated, quantized, scale = residual_rms_norm_quantized(
        state["x"], state["branch"], state["weight"], EPS, dtype=state["dtype"],
        group_size=state["group"])
    if state["dtype"] == torch.int8:
        quantized = dequantize(quantized, scale, group_size=state["group"], dtype=torch.bfloat16)
    return updated, quantized, scale


def _own_step(state):
    from gfx1010_kernels import residual_rms_norm

    updated, normalized = residual_rms_norm(
        state["x"], state["branch"], state["weight"], EPS, normalized_dtype=state["dtype"],
        checkpoint_dtype=state["checkpoint"])
    gradients = torch.autograd.grad(
        [updated, normalized], [state["x"], state["branch"], state["weight"]],
        [state["grad_updated"], state["grad_normalized"]])
    return (updated, normalized, *gradients)


def run(state):
    if state["kind"] == "step":
        if own:
            return _own_step(state)
        with torch.no_grad():
            return _plain_step(state)
    with torch.no_grad():
        if state["kind"] == "quant":
            return _own_quantized(state) if own else _plain_quantized(state)
        return _own_call(state) if own else _plain_call(state)


def work(case):
    """Compulsory traffic: every input read once, every output written once,
    what a training forward keeps for its backward written and read once."""
    hidden = case["hidden"]
    rows = case["batch"] * case["length"]
    count = rows * hidden
    x, branch, normalized = SIZES[case["x"]], SIZES[case["branch"]], SIZES[case["normalized"]]
    weight = hidden * SIZES[case["weight"]]
    total = count * (x + branch + x + normalized) + weight
    flops = 8.0 * count
    if case["kind"] == "quant":
        groups = rows * (-(-hidden // case["group"]) if case["group"] else 1)
        total += 4 * groups
        if case["normalized"] == "int8":  # read again and widened to bf16
            total += 4 * groups + 3 * count
            flops += count
    elif case["kind"] == "step":
        # the kept input and both upstream gradients -> grad_x, grad_branch, grad_weight
        kept = x * count
        if case["checkpoint"]:
            kept = count + 4 * rows * -(-hidden // CHECKPOINT_GROUP)
            total += kept
        total += kept + count * (x + normalized + x) + 2 * weight + 2 * 4 * rows
        if case["branch"] != case["x"]:
            total += branch * count
        flops += 14.0 * count
    return {"bytes": total, "flops": flops}


def exact(case, seed):
    inputs = _inputs(case, seed)
    hidden, rows = case["hidden"], case["batch"] * case["length"]
    shape = (case["batch"], case["length"])
    weight = inputs["weight"].double()
    group = CHECKPOINT_GROUP if case["checkpoint"] else case["group"] or hidden
    groups = -(-hidden // group)
    dtype = DTYPES[case["normalized"]]
    top = 127.0 if case["checkpoint"] else TOP.get(dtype)

    def eight_bits(values):
        """Whole steps of each value (fp32 values as float64) and each group's
        maximum; each quotient and product is rounded to fp32 once."""
        largest = torch.stack([part.abs().amax(-1) for part in values.split(group, -1)], -1)
        largest = largest.clamp(min=TINY)
        inverse = (top / largest).float().double()
        where = torch.arange(hidden, device="cuda") // group
        return (values * inverse[:, where]).float(), largest, where

    def piece(a, b):
        x, branch = inputs["x"].reshape(rows, hidden)[a:b], inputs["branch"].reshape(rows, hidden)
        updated = (x.double() + branch[a:b].double()).to(x.dtype).double()
        rstd = (updated.square().mean(-1, keepdim=True) + EPS).rsqrt()
        if case["kind"] == "quant":
            steps, largest, where = eight_bits((updated * weight).float().double())
            scale = largest / top * rstd
            if dtype == torch.int8:
                return updated, steps.double().round() * scale[:, where], scale
            return updated, steps.to(dtype).double(), scale
        normalized = updated * rstd * weight
        if case["kind"] == "call":
            return updated, normalized
        kept = updated
        if case["checkpoint"]:
            steps, largest, where = eight_bits(updated)
            kept = steps.double().round() * (largest / top).float().double()[:, where]
        upstream = inputs["grad_normalized"].reshape(rows, hidden)[a:b].double()
        unit, product = kept * rstd, upstream * weight
        gradient = inputs["grad_updated"].reshape(rows, hidden)[a:b].double() + rstd * (
            product - unit * (product * unit).mean(-1, keepdim=True))
        return updated, normalized, gradient, gradient, (upstream * unit).sum(0, keepdim=True)

    step = max(1, (1 << 23) // hidden)
    parts = [piece(a, min(rows, a + step)) for a in range(0, rows, step)]
    answer = []
    for index, column in enumerate(zip(*parts)):
        if index == 4:
            answer.append(torch.cat(column).sum(0))
        else:
            whole = torch.cat(column)
            answer.append(whole.view(*shape, whole.shape[-1]))
    return tuple(answer)
