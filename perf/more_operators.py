"""The operators of a model served in 8-bit integers, on their own: the product of rows and weights held as 8-bit integers with a
scale per token and per output channel, and what makes such rows: the norm (with the residual's addition), the gated unit, and a
plain rounding of rows.

A case is one call.  The widths are those of the engine's own models (1,024, 4,096 and 5,120 wide, feed-forwards of 12,288 and
25,600) and generic ones; the numbers of tokens are those of a decode step, of a prompt and of a large portion.

``run`` computes the formulas with elementary torch operations in 32 bits, or, where ``own`` is set, calls the engine's kernels.
8-bit rows are returned as the values they stand for (integer times scale), in 16 bits.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


# ------------------------------------------------------------------------------------------------ the cases
def _product(name, tokens, k, n, out="bf16", pitch=16):
    """``pitch``: the rows of both operands start at multiples of that many bytes (1: packed without gaps)."""
    return {"name": name, "op": "product", "tokens": tokens, "k": k, "n": n, "out": out, "pitch": pitch}


def _rows(name, op, rows, width, dtype="bf16", residual=False):
    return {"name": name, "op": op, "rows": rows, "width": width, "dtype": dtype, "residual": residual}


def listed():
    return [
        # one token through the output projection of the attention of a small model: latency is all there is
        _product("product_token_1", 1, 2048, 1024),
        # a decode step of 8 requests, gate and up projections of the 8B-shaped model: the weights are read once
        _product("product_decode_8", 8, 4096, 24576),
        # a decode step of 64 requests, the down projection
        _product("product_decode_64", 64, 12288, 4096),
        # a prompt of 2,048 tokens, gate and up projections
        _product("product_prompt_2048", 2048, 4096, 24576),
        # a full step of prompt portions through the q, k and v projections of the 32B-shaped model
        _product("product_portion_8192", 8192, 5120, 10240),
        # a mixed step of a model whose widths divide by little, output in 32 bits
        _product("product_odd_333", 333, 1001, 2774, out="f32"),
        # the norm in front of a sub-block, with the residual's addition: a decode step and a step of prompt portions
        _rows("norm_decode_8", "norm", 8, 4096, residual=True),
        _rows("norm_portion_8191", "norm", 8191, 5120, residual=True),
        # the gated unit between the feed-forward's two products: a decode step and a prompt
        _rows("unit_decode_8", "unit", 8, 12288),
        _rows("unit_prompt_2048", "unit", 2048, 25600),
        # what the attention returns, in front of its output projection; and a weight matrix as it is loaded, row by row
        _rows("round_decode_64", "round", 64, 4096),
        _rows("round_weights", "round", 24576, 4096),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))


def _width(rng, lo, hi):
    """A width of a layer: most divide by 64 or 128, some by 8, some by nothing."""
    w = _log(rng, lo, hi)
    step = rng.choice((128, 128, 64, 8, 1))
    return max(step, w // step * step)


def draw(rng):
    if rng.random() < 0.5:
        tokens = _log(rng, 1, 64) if rng.random() < 0.5 else _log(rng, 65, 8192)
        k, n = _width(rng, 64, 25600), _width(rng, 64, 50000)
        out = rng.choice(("bf16", "bf16", "bf16", "f32"))
        # no dearer than the largest listed cases, in operations and in bytes
        while tokens * k * n > 1 << 38 or tokens * n > 1 << (26 if out == "bf16" else 25) or k * n > 1 << 27:
            tokens, k, n = max(1, tokens * 3 // 4), k if k < n else max(64, k // 2), n if n < k else max(64, n // 2)
        case = _product("", tokens, k, n, out, rng.choice((16, 16, 16, 128, 1)))
    else:
        op = rng.choice(("norm", "norm", "unit", "round"))
        rows = _log(rng, 1, 64) if rng.random() < 0.4 else _log(rng, 65, 16384)
        width = _width(rng, 33, 25600)
        dtype = rng.choice(("bf16", "bf16", "bf16", "f32"))
        while rows * width > 1 << (25 if dtype == "bf16" else 24):
            rows = max(1, rows // 2)
        case = _rows("", op, rows, width, dtype, op == "norm" and rng.random() < 0.7)
    del case["name"]
    return case


def work(case):
    if case["op"] == "product":
        t, k, n = case["tokens"], case["k"], case["n"]
        return {"bytes": t * k + n * k + 4 * (t + n) + t * n * (2 if case["out"] == "bf16" else 4), "flops": 2 * t * k * n}
    r, w, item = case["rows"], case["width"], 2 if case["dtype"] == "bf16" else 4
    read = w * item * {"norm": 3 if case["residual"] else 1, "unit": 2, "round": 1}[case["op"]]    # the residual: read and written
    return {"bytes": r * (read + w + 4) + (w * item if case["op"] == "norm" else 0), "flops": r * w * {"norm": 8, "unit": 10, "round": 4}[case["op"]]}


# ------------------------------------------------------------------------------------------------ what a program has in hand
def _eight_bits(x):
    """Rows [n, w] as 8-bit integers and a scale each."""
    top = x.float().abs().amax(1, keepdim=True)
    safe = torch.where(top == 0, 1.0, top)
    return torch.round(x.float() * 127 / safe).to(torch.int8), (top / 127)[:, 0].contiguous()


def _pitched(q, pitch):
    rows, width = q.shape
    full = torch.zeros((rows, -(-width // pitch) * pitch), dtype=torch.int8, device=q.device)
    full[:, :width] = q
    return full[:, :width]


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    normal = lambda *shape: torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)      # noqa: E731
    if case["op"] == "product":
        x = normal(case["tokens"], case["k"])
        x *= torch.exp(0.6 * normal(1, case["k"]))              # some channels carry much more than others
        q, scales = _eight_bits(x)
        w, w_scales = _eight_bits(normal(case["n"], case["k"]) * (0.02 * torch.exp(0.3 * normal(case["n"], 1))))
        return {"case": case, "x": _pitched(q, case["pitch"]), "x_scales": scales, "w": _pitched(w, case["pitch"]), "w_scales": w_scales}
    dt, rows, width = DTYPES[case["dtype"]], case["rows"], case["width"]
    state = {"case": case}
    if case["op"] == "unit":
        state["gate_up"] = (normal(rows, 2 * width) * 1.3).to(dt)
        return state
    state["x"] = (normal(rows, width) * torch.exp(0.5 * normal(1, width))).to(dt)
    if case["op"] == "norm":
        state["weight"] = (1.0 + 0.2 * normal(width)).to(dt)
        if case["residual"]:
            state["residual"] = (3.0 * normal(rows, width)).to(dt)
    return state


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    case = state["case"]
    if own:
        return _own(state)
    if case["op"] == "product":
        total = state["x"].float() @ state["w"].float().t()
        return {"out": (total * state["x_scales"][:, None] * state["w_scales"][None]).to(DTYPES[case["out"]])}
    if case["op"] == "unit":
        gate, up = state["gate_up"].float().split(case["width"], 1)
        return _plain_rows(gate / (1 + torch.exp(-gate)) * up)
    x = state["x"].float()
    if case["op"] == "round":
        return _plain_rows(x)
    if case["residual"]:
        x = x + state["residual"].float()
        state["residual"].copy_(x)                              # rounded to the model's type once
    y = x * torch.rsqrt((x * x).mean(1, keepdim=True) + EPS) * state["weight"].float()
    out = _plain_rows(y)
    if case["residual"]:
        out["residual"] = state["residual"]
    return out


EPS = 1e-6


def _plain_rows(y):
    top = y.abs().amax(1, keepdim=True)
    q = torch.round(y * 127 / torch.where(top == 0, 1.0, top))
    scales = top / 127
    return {"values": (q * scales).to(torch.bfloat16), "scales": scales[:, 0]}


def _own(state):
    from nanohybrid_vlm_b200.kernels import ops
    case = state["case"]
    if case["op"] == "product":
        out = torch.empty((case["tokens"], case["n"]), dtype=DTYPES[case["out"]], device="cuda")
        ops.linear_int8(out, state["x"], state["x_scales"], state["w"], state["w_scales"])
        return {"out": out}
    q = ops.new_int8(case["rows"], case["width"], "cuda")
    scales = torch.empty(case["rows"], dtype=torch.float32, device="cuda")
    if case["op"] == "norm":
        ops.rmsnorm_int8(q, scales, state["x"], state["weight"], EPS, residual=state.get("residual"))
    elif case["op"] == "unit":
        ops.silu_mul_int8(q, scales, state["gate_up"])
    else:
        ops.quantize_rows(q, scales, state["x"])
    values = torch.empty((case["rows"], case["width"]), dtype=torch.bfloat16, device="cuda")
    ops.dequantize_rows(values, q, scales)
    out = {"values": values, "scales": scales}
    if case["residual"]:
        out["residual"] = state["residual"]
    return out


# ------------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    """The definitions in 64 bits, a block of rows at a time."""
    state = prepare(case, seed)
    if case["op"] == "product":
        w = state["w"].double() * state["w_scales"].double()[:, None]
        return {"out": torch.cat([(x.double() * s.double()[:, None]) @ w.T
                                  for x, s in zip(state["x"].split(2048), state["x_scales"].split(2048))])}
    given = state["gate_up"] if case["op"] == "unit" else state["x"]
    values, scales, sums = [], [], []
    for i in range(0, case["rows"], 2048):
        y = given[i:i + 2048].double()
        if case["op"] == "unit":
            y = torch.sigmoid(y[:, :case["width"]]) * y[:, :case["width"]] * y[:, case["width"]:]
        elif case["op"] == "norm":
            if case["residual"]:
                y = y + state["residual"][i:i + 2048].double()
                sums.append(y)
            y = y / torch.sqrt(y.pow(2).mean(dim=1, keepdim=True) + EPS) * state["weight"].double()
        step = y.abs().max(dim=1).values / 127.0
        scales.append(step)
        step = step.unsqueeze(1)
        values.append(torch.where(step > 0, torch.round(y / step.clamp(min=1e-300)) * step, 0.0))
    out = {"values": torch.cat(values), "scales": torch.cat(scales)}
    if case["residual"]:
        out["residual"] = torch.cat(sums)
    return out
