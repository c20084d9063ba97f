"""Timed cases of the operators around an expert feed-forward layer: the residual addition and RMSNorm with an 8-bit output,
the gated activation that keeps its input in 8 bits for the backward pass, and the matrix products grouped by expert.

``run`` makes one call of one operator.  With ``own`` set it calls ``taac_2026_b200.ops``; without it the operator is computed
from elementary torch operations in 32 bits and rounded once.  ``exact`` computes the same values in 64 bits.
"""

import math
import random

import numpy as np
import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
EPS = 1e-6
BLOCK = 128         # values that share a scale
E4M3_MAX = 448.0


def listed():
    return [
        # one request's token ahead of an e4m3 feed-forward layer of width 512: latency
        {"name": "norm quant one row", "op": "norm_quant", "rows": 1, "cols": 512, "type": "bf16"},
        # all tokens of a training or scoring batch at the model's width
        {"name": "norm quant 262144 x 512", "op": "norm_quant", "rows": 262144, "cols": 512, "type": "bf16"},
        # a wide tokenizer's rows (2560 = 20 fields of 128), a batch whose rows fill no tile
        {"name": "norm quant 5003 x 2560", "op": "norm_quant", "rows": 5003, "cols": 2560, "type": "fp16"},
        # the training step's backward pass at the model's width
        {"name": "norm backward 65536 x 512", "op": "norm_backward", "rows": 65536, "cols": 512, "type": "bf16"},
        # parity training in full precision on wide rows, few of them
        {"name": "norm backward 1201 x 4096", "op": "norm_backward", "rows": 1201, "cols": 4096, "type": "fp32"},
        # gated layer of 512 -> 2 x 2048: the activation of a training batch and what it keeps
        {"name": "gate 32768 x 2048", "op": "gate", "rows": 32768, "hidden": 2048, "gated": True, "type": "bf16"},
        # its backward pass from the kept 8 bits
        {"name": "gate backward 32768 x 2048", "op": "gate_backward", "rows": 32768, "hidden": 2048, "gated": True, "type": "bf16"},
        # a small ungated layer, ragged rows
        {"name": "gate backward 777 x 640", "op": "gate_backward", "rows": 777, "hidden": 640, "gated": False, "type": "fp16"},
        # a few requests' tokens routed over sixteen experts: the weights are the traffic
        {"name": "experts 24 rows", "op": "experts", "rows": 24, "experts": 16, "k": 512, "n": 2048, "silu": True, "type": "bf16"},
        # a training batch through the up projections of nine parameter groups
        {"name": "experts 65536 rows", "op": "experts", "rows": 65536, "experts": 9, "k": 512, "n": 2048, "silu": False, "type": "bf16"},
        # gradients of rows, weights and biases of such a layer
        {"name": "experts backward 32768 rows", "op": "experts_backward", "rows": 32768, "experts": 16, "k": 512, "n": 2048, "type": "bf16"},
        # odd widths and ragged groups, some of them empty
        {"name": "experts backward 1999 rows", "op": "experts_backward", "rows": 1999, "experts": 12, "k": 520, "n": 1000, "type": "fp16"},
    ]


def _log(rng, lo, hi, step=1):
    """A multiple of `step` in [lo, hi], spread over the logarithm."""
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi)))) // step * step))


def draw(rng):
    op = rng.choice(["norm_quant", "norm_backward", "gate", "gate_backward", "experts", "experts_backward"])
    if op in ("norm_quant", "norm_backward"):
        # one row to a large batch, 128 to 8192 columns, at most 2^26 values
        cols = _log(rng, 128, 8192, 128)
        return {"op": op, "rows": _log(rng, 1, min(262144, (1 << 26) // cols)), "cols": cols, "type": rng.choice(["bf16", "fp16", "fp32"])}
    if op in ("gate", "gate_backward"):
        hidden = _log(rng, 128, 8192, 128)
        return {"op": op, "rows": _log(rng, 1, min(65536, (1 << 25) // hidden)), "hidden": hidden, "gated": rng.random() < 0.7,
                "type": rng.choice(["bf16", "fp16", "fp32"])}
    # one row to a training batch, 1 to 64 experts, widths in whole 16-byte pieces; at most 2^34 products a direction
    k, n, experts = _log(rng, 64, 2048, 8), _log(rng, 64, 2048, 8), _log(rng, 1, 64)
    case = {"op": op, "rows": _log(rng, 1, min(65536, (1 << 34) // (k * n))), "experts": experts, "k": k, "n": n, "type": rng.choice(["bf16", "fp16"])}
    return {**case, "silu": rng.random() < 0.5} if op == "experts" else case


def group_sizes(case):
    """Rows of each expert: uneven by up to a factor of three around the mean, some experts without rows."""
    rng = random.Random(case["rows"] * 1009 + case["experts"])
    share = [0.0 if rng.random() < 0.1 else rng.uniform(0.5, 1.5) for _ in range(case["experts"])]
    if not any(share):
        share[-1] = 1.0
    ends = [int(round(case["rows"] * s / sum(share))) for s in np.cumsum(share)]
    return [e - b for b, e in zip([0] + ends[:-1], ends)]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = TYPES[case["type"]]

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(dtype)

    state = {"op": case["op"], "case": case, "dtype": dtype}
    if case["op"] in ("norm_quant", "norm_backward"):
        rows, cols = case["rows"], case["cols"]
        state["weight"] = 1 + normal(cols, scale=0.1)
        if case["op"] == "norm_quant":
            state["x"], state["residual"] = normal(rows, cols), normal(rows, cols, scale=2.0)
        else:
            state["total"], state["grad_normed"], state["grad_total"] = normal(rows, cols, scale=2.0), normal(rows, cols), normal(rows, cols)
    elif case["op"] in ("gate", "gate_backward"):
        rows, hidden, width = case["rows"], case["hidden"], case["hidden"] * (2 if case["gated"] else 1)
        up = normal(rows, width, scale=2.0)
        if case["op"] == "gate":
            state["up"] = up
        else:
            # what the forward pass kept: e4m3 values and a power of two for each 128 of them
            state["q"], state["scales"] = _kept(up)
            state["grad"] = normal(rows, hidden)
    else:
        sizes = group_sizes(case)
        state["cap"] = max(sizes)     # rows of the largest group, as a program that pads groups keeps it
        state["offsets"] = torch.tensor([0] + list(np.cumsum(sizes)), dtype=torch.int32, device="cuda")
        state["x"] = normal(case["rows"], case["k"])
        state["weight"] = normal(case["experts"], case["n"], case["k"], scale=case["k"] ** -0.5)
        if case["op"] == "experts":
            state["bias"] = torch.randn(case["experts"], case["n"], generator=gen, device="cuda") * 0.1
        else:
            state["grad"] = normal(case["rows"], case["n"])
    return state


# ---------------------------------------------------------------------------------------------- plain forms
def _kept(x):
    """e4m3 values of x [rows, width] and a power of two for each 128 of them: the smallest with |x| / scale <= 448."""
    blocks = x.float().reshape(x.shape[0], -1, BLOCK)
    amax = blocks.abs().amax(-1)
    mantissa, exponent = torch.frexp(amax)      # 448 = 0.875 * 2^9: compared without a rounding
    exponent = exponent - 9 + (mantissa > 0.875)
    scales = torch.where(amax > 0, torch.ldexp(torch.ones_like(amax), exponent.clamp(-126, 126)), torch.ones_like(amax))
    q = (blocks / scales[..., None]).to(torch.float8_e4m3fn)
    return q.reshape(x.shape), scales


def _norm_quant(x, residual, weight):
    s = x.float() + residual.float()
    normed = s * torch.rsqrt((s * s).mean(-1, keepdim=True) + EPS) * weight.float()
    blocks = normed.reshape(s.shape[0], -1, BLOCK)
    amax = blocks.abs().amax(-1)
    scales = torch.where(amax > 0, amax / E4M3_MAX, torch.ones_like(amax))
    q = (blocks / scales[..., None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
    return s.to(x.dtype), q.reshape(s.shape), scales


def _norm_backward(total, weight, grad_normed, grad_total):
    s, dy = total.float(), grad_normed.float()
    r = torch.rsqrt((s * s).mean(-1, keepdim=True) + EPS)
    xh, g = s * r, dy * weight.float()
    grad = r * (g - xh * (g * xh).mean(-1, keepdim=True)) + grad_total.float()
    # the sum over all rows is long: 64 bits
    return grad.to(total.dtype), (dy * xh).sum(0, dtype=torch.float64).to(weight.dtype)


def _gate(up, gated):
    u = up.float()
    gate, value = u.chunk(2, -1) if gated else (u, None)
    h = gate * torch.sigmoid(gate)
    q, scales = _kept(up)
    return (h if value is None else h * value).to(up.dtype), q, scales


def _gate_backward(q, scales, grad, gated):
    u = (q.float().reshape(q.shape[0], -1, BLOCK) * scales[..., None]).reshape(q.shape)
    gate, value = u.chunk(2, -1) if gated else (u, None)
    sig, dh = torch.sigmoid(gate), grad.float()
    silu = gate * sig
    slope = sig * (1 + gate * (1 - sig))
    if value is None:
        return (dh * slope).to(grad.dtype), silu.to(grad.dtype)
    return torch.cat([dh * value * slope, dh * silu], -1).to(grad.dtype), (silu * value).to(grad.dtype)


def _padded(state):
    """Row numbers [experts, cap] of each group, and which of them are rows of the group."""
    begin, end = state["offsets"][:-1].long(), state["offsets"][1:].long()
    index = begin[:, None] + torch.arange(state["cap"], device="cuda")
    return index.clamp(max=state["x"].shape[0] - 1), index < end[:, None]


def _experts(state, silu):
    index, inside = _padded(state)
    y = torch.bmm(state["x"].float()[index], state["weight"].float().transpose(1, 2)) + state["bias"][:, None]
    if silu:
        y = y * torch.sigmoid(y)
    out = torch.zeros(state["x"].shape[0], y.shape[-1], device="cuda")
    out[index[inside]] = y[inside]
    return out.to(state["dtype"])


def _experts_backward(state):
    index, inside = _padded(state)
    x = torch.where(inside[..., None], state["x"].float()[index], 0.0)
    dy = torch.where(inside[..., None], state["grad"].float()[index], 0.0)
    dx = torch.zeros(state["x"].shape, device="cuda")
    dx[index[inside]] = torch.bmm(dy, state["weight"].float())[inside]
    dw = torch.bmm(dy.transpose(1, 2), x)
    return dx.to(state["dtype"]), dw.to(state["dtype"]), dy.sum(1)


def run(state):
    op, case = state["op"], state["case"]
    if own:
        from taac_2026_b200 import ops

        if op == "norm_quant":
            return ops.add_rms_norm_quant(state["x"], state["residual"], state["weight"], EPS)
        if op == "norm_backward":
            return ops.add_rms_norm_backward(state["total"], state["weight"], state["grad_normed"], state["grad_total"], EPS)
        if op == "gate":
            return ops.silu_gate_checkpoint(state["up"], gated=case["gated"])
        if op == "gate_backward":
            return ops.silu_gate_backward(state["q"], state["scales"], state["grad"], gated=case["gated"])
        if op == "experts":
            return ops.ragged_linear(state["x"], state["weight"], state["offsets"], state["bias"], silu=case["silu"])
        return ops.ragged_linear_backward(state["x"], state["weight"], state["offsets"], state["grad"], bias=True)
    if op == "norm_quant":
        return _norm_quant(state["x"], state["residual"], state["weight"])
    if op == "norm_backward":
        return _norm_backward(state["total"], state["weight"], state["grad_normed"], state["grad_total"])
    if op == "gate":
        return _gate(state["up"], case["gated"])
    if op == "gate_backward":
        return _gate_backward(state["q"], state["scales"], state["grad"], case["gated"])
    if op == "experts":
        return _experts(state, case["silu"])
    return _experts_backward(state)


def work(case):
    op, e = case["op"], SIZE[case["type"]]
    if op in ("norm_quant", "norm_backward"):
        rows, cols = case["rows"], case["cols"]
        if op == "norm_quant":      # x, residual -> total, 8-bit values, scales
            return {"bytes": rows * cols * (3 * e + 1) + rows * cols // BLOCK * 4 + cols * e, "flops": 6 * rows * cols}
        return {"bytes": rows * cols * 4 * e + 2 * cols * e, "flops": 10 * rows * cols}
    if op in ("gate", "gate_backward"):
        rows, hidden, width = case["rows"], case["hidden"], case["hidden"] * (2 if case["gated"] else 1)
        kept = rows * width + rows * width // BLOCK * 4
        if op == "gate":            # input -> activation, 8-bit values, scales
            return {"bytes": rows * (width + hidden) * e + kept, "flops": 8 * rows * hidden}
        # 8-bit values, gradient -> gradient of the input, the activation again for the next layer's weight gradient
        return {"bytes": kept + rows * (2 * hidden + width) * e, "flops": 12 * rows * hidden}
    rows, k, n, experts = case["rows"], case["k"], case["n"], case["experts"]
    active = sum(s > 0 for s in group_sizes(case))
    if op == "experts":
        return {"bytes": rows * (k + n) * e + active * n * (k * e + 4) + 4 * (experts + 1), "flops": 2 * rows * k * n}
    # x, gradient, weights -> gradients of rows, weights (all experts', zeros among them) and biases
    return {"bytes": rows * (2 * k + n) * e + (active + experts) * n * k * e + experts * n * 4 + 4 * (experts + 1), "flops": 4 * rows * k * n}


# ---------------------------------------------------------------------------------------------- 64 bits
def _silu64(z):
    return z / (1 + torch.exp(-z))


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "norm_quant":
        t = s["x"].double() + s["residual"].double()
        y = t / torch.sqrt(t.pow(2).sum(1, keepdim=True) / t.shape[1] + EPS) * s["weight"].double()
        top = y.view(t.shape[0], -1, BLOCK).abs().max(2).values / E4M3_MAX
        return t, y / top.repeat_interleave(BLOCK, 1), top
    if op == "norm_backward":
        t, w, dy = s["total"].double(), s["weight"].double(), s["grad_normed"].double()
        ms = t.pow(2).sum(1, keepdim=True) / t.shape[1] + EPS
        dot = (dy * w * t).sum(1, keepdim=True) / t.shape[1]
        return dy * w / ms.sqrt() - t * dot / ms.pow(1.5) + s["grad_total"].double(), (dy * t / ms.sqrt()).sum(0)
    if op == "gate":
        u, n = s["up"].double(), case["hidden"]
        amax = u.view(u.shape[0], -1, BLOCK).abs().max(2).values
        mantissa, exponent = torch.frexp(amax / E4M3_MAX)      # the power of two itself has the mantissa 0.5
        scales = torch.where(mantissa == 0.5, 0.5, 1.0).double() * torch.exp2(exponent.double())
        return _silu64(u[:, :n]) * (u[:, n:] if case["gated"] else 1), u / scales.repeat_interleave(BLOCK, 1), scales
    if op == "gate_backward":
        n, dh = case["hidden"], s["grad"].double()
        u = s["q"].double() * s["scales"].double().repeat_interleave(BLOCK, 1)
        g, v = u[:, :n], (u[:, n:] if case["gated"] else torch.ones_like(u))
        p = 1 / (1 + torch.exp(-g))
        dg = dh * v * (p + g * p * torch.exp(-g) / (1 + torch.exp(-g)))
        return (torch.cat([dg, dh * _silu64(g)], 1) if case["gated"] else dg), _silu64(g) * v
    sizes = group_sizes(case)
    x, w = s["x"].double().split(sizes), s["weight"].double()
    if op == "experts":
        y = torch.cat([xe @ we.T + be for xe, we, be in zip(x, w, s["bias"].double())])
        return _silu64(y) if case["silu"] else y
    dy = s["grad"].double().split(sizes)
    return (torch.cat([g @ we for g, we in zip(dy, w)]), torch.stack([g.T @ xe for g, xe in zip(dy, x)]), torch.stack([g.sum(0) for g in dy]))
