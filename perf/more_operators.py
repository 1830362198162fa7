"""Operators of an expert block that is trained, and of one that is served in 8 bits, as measurable cases: projections and expert layers on
8-bit integers with a scale for each token and each channel (``int8.linear_int8``, ``int8.moe_forward_int8``), tokens sorted by expert and
back with the router's weights (``moe_train.route``, ``sort_rows``, ``combine_rows``), the activation between an expert's products
(``moe_train.gated``), dropout whose mask is never stored (``dropout.dropout``); the last three with their gradients.

``own`` false: the operators in their plain form, elementary torch operations in 32 bits, rounded once at the end.  ``own`` true: the
calls that a user of the package makes.  Ranges that the listed cases stand for:

    projections    1 to 8192 tokens, inner and outer size 64 to 16384, odd ones too; bf16, fp16 and fp32 activations
    expert layers  1 to 4096 tokens, 4 to 128 experts, 1 to 8 choices, hidden size 256 to 4096, inner size 128 to 14336, weights up to
                   1.5 GB; bf16 and fp16; SwiGLU and SiLU
    sorting        1 to 32768 tokens, 4 to 256 experts, 1 to 8 choices, rows of 64 to 8192 elements; bf16, fp16, fp32; weights over the
                   chosen experts or over all
    activation     1 to 65536 rows, inner size 64 to 14336; SwiGLU and SiLU; bf16, fp16, fp32; rows that lie apart
    dropout        1 to 65536 rows of 64 to 16384 elements; bf16, fp16, fp32; with and without a residual; rows that lie apart
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEVICE = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
SMALLEST = 2.0 ** -100     # rows and columns of 8-bit matrices whose largest element is below it are held as zeros
MAX_LINEAR_FLOPS = 1e12    # a drawn case costs no more than the largest listed one
MAX_LAYER_BYTES = 1.5e9
MAX_LAYER_FLOPS = 4e11
MAX_SORT_ELEMENTS = 2.7e8
MAX_GATED_ELEMENTS = 2.4e8
MAX_DROPOUT_ELEMENTS = 6.8e7


# ---------------------------------------------------------------------------------------------- cases
def _linear(tokens, inner, outer, dtype="bf16"):
    return {"op": "linear", "T": tokens, "K": inner, "N": outer, "dtype": dtype}


def _layer(tokens, experts, top_k, hidden, inner, kind="swiglu", dtype="bf16"):
    return {"op": "layer", "T": tokens, "E": experts, "top_k": top_k, "H": hidden, "I": inner, "kind": kind, "dtype": dtype}


def _sort(tokens, experts, top_k, hidden, dtype="bf16", logits="fp32", renormalize=True):
    return {"op": "sort", "T": tokens, "E": experts, "top_k": top_k, "H": hidden, "dtype": dtype, "logits": logits, "renormalize": renormalize}


def _gated(rows, inner, kind="swiglu", dtype="bf16", pad=0):
    """pad: the rows of the activation's operand lie that much further apart."""
    return {"op": "gated", "rows": rows, "I": inner, "kind": kind, "dtype": dtype, "pad": pad}


def _dropout(rows, width, p, residual=True, dtype="bf16", pad=0):
    """pad: the rows of the operand lie that much further apart."""
    return {"op": "dropout", "rows": rows, "width": width, "p": p, "residual": residual, "dtype": dtype, "pad": pad}


def listed():
    cases = {
        # one sequence is being answered: a block's output projection, latency alone
        "int8_one": _linear(1, 4096, 4096),
        # a decoding step of 48 sequences through a wide projection
        "int8_decode": _linear(48, 4096, 14336),
        # a batch of prompts through a wide projection
        "int8_prefill": _linear(8192, 4096, 14336),
        # one token through many small experts: latency
        "int8_layer_one": _layer(1, 128, 8, 2048, 768),
        # a decoding step of 24 sequences through few large experts, half precision
        "int8_layer_decode": _layer(24, 8, 2, 4096, 14336, dtype="fp16"),
        # a batch of prompts, no round number of tokens, through many small experts
        "int8_layer_prefill": _layer(4001, 128, 8, 2048, 768),
        # a few tokens of odd width, weights over all experts, half precision: latency of both directions
        "sort_odd": _sort(61, 60, 4, 1031, dtype="fp16", logits="fp16", renormalize=False),
        # a training step's tokens to many small experts and back
        "sort_train": _sort(16384, 128, 8, 2048),
        # full precision, odd width, rows that lie apart
        "gated_odd": _gated(1003, 1031, dtype="fp32", pad=5),
        # a training step's activations in large experts
        "gated_train": _gated(16384, 14336),
        # a short batch, half precision: latency of both directions
        "dropout_small": _dropout(129, 2048, 0.1, dtype="fp16"),
        # the residual stream of a training step
        "dropout_train": _dropout(16384, 4096, 0.1),
    }
    return [dict(case, name=name) for name, case in cases.items()]


def _log(rng, lo, hi):
    """Whole number between lo and hi, uniform in its logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _draw_linear(rng):
    inner, outer = _log(rng, 64, 16384), _log(rng, 64, 16384)
    if rng.random() < 0.7:
        inner, outer = inner // 16 * 16, outer // 8 * 8
    return _linear(_log(rng, 1, 128) if rng.random() < 0.4 else _log(rng, 1, 8192), inner, outer, dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]))


def _draw_layer(rng):
    experts = _log(rng, 4, 128)
    hidden, inner = _log(rng, 256, 4096), _log(rng, 128, 14336)
    if rng.random() < 0.8:
        hidden, inner = hidden // 16 * 16, inner // 16 * 16
    return _layer(_log(rng, 1, 64) if rng.random() < 0.5 else _log(rng, 1, 4096), experts, rng.randint(1, min(8, experts)), hidden, inner,
                  kind=rng.choice(["swiglu", "swiglu", "silu"]), dtype=rng.choice(["bf16", "bf16", "fp16"]))


def _draw_sort(rng):
    experts, hidden = _log(rng, 4, 256), _log(rng, 64, 8192)
    if rng.random() < 0.7:
        hidden = hidden // 8 * 8
    return _sort(_log(rng, 1, 32768), experts, rng.randint(1, min(8, experts)), hidden, dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                 logits=rng.choice(["fp32", "bf16", "fp16"]), renormalize=rng.random() < 0.6)


def _draw_gated(rng):
    inner = _log(rng, 64, 14336)
    if rng.random() < 0.7:
        inner = inner // 8 * 8
    return _gated(_log(rng, 1, 65536), inner, kind=rng.choice(["swiglu", "swiglu", "silu"]), dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                  pad=rng.choice([0, 0, 8, 3]))


def _draw_dropout(rng):
    return _dropout(_log(rng, 1, 65536), _log(rng, 64, 16384), rng.choice([0.1, 0.1, 0.05, 0.3, 0.5]), residual=rng.random() < 0.6,
                    dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]), pad=rng.choice([0, 0, 8, 3]))


def draw(rng):
    while True:
        case = rng.choice([_draw_linear, _draw_linear, _draw_layer, _draw_layer, _draw_sort, _draw_gated, _draw_dropout])(rng)
        if case["op"] == "linear" and work(case)["flops"] <= MAX_LINEAR_FLOPS:
            return case
        if case["op"] == "layer" and case["E"] * _weights(case) <= MAX_LAYER_BYTES and work(case)["flops"] <= MAX_LAYER_FLOPS:
            return case
        if case["op"] == "sort" and case["T"] * case["top_k"] * case["H"] <= MAX_SORT_ELEMENTS * (0.5 if case["dtype"] == "fp32" else 1.0):
            return case
        if case["op"] == "gated" and case["rows"] * case["I"] <= MAX_GATED_ELEMENTS * (0.5 if case["dtype"] == "fp32" else 1.0):
            return case
        if case["op"] == "dropout" and case["rows"] * case["width"] <= MAX_DROPOUT_ELEMENTS:
            return case


def _weights(case):
    """Elements of one expert's two matrices."""
    return case["H"] * case["I"] * (2 if case["kind"] == "silu" else 3)


# ---------------------------------------------------------------------------------------------- inputs
def _random(gen, shape, dtype, scale=1.0):
    t = torch.randn(shape, device=DEVICE, dtype=dtype, generator=gen)
    return t if scale == 1.0 else t.mul_(scale)


def _rows(gen, rows, width, pad, dtype):
    """Rows of `width` elements that lie width + pad apart."""
    return _random(gen, (rows, width + pad), dtype)[:, :width]


def _matrix(gen, shape):
    """A (stack of) 8-bit matrices [.., K, N], contiguous along K as a linear layer stores them, their columns 16-byte aligned, and a scale for
    each column: normal weights of variance 1 / K, whose columns' largest elements lie around 3.5 deviations."""
    *batch, K, N = shape
    values = torch.randn((*batch, N, -(-K // 16) * 16), device=DEVICE, dtype=torch.bfloat16, generator=gen).mul_(127 / 3.5).round_().clamp_(-127, 127)
    scale = (0.9 + 0.2 * torch.rand((*batch, N), device=DEVICE, generator=gen)) * (3.5 / 127 * K ** -0.5)
    return values.to(torch.int8)[..., :K].transpose(-2, -1), scale


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    op = case["op"]
    if op == "linear":
        values, scale = _matrix(gen, (case["K"], case["N"]))
        return {"op": op, "x": _random(gen, (case["T"], case["K"]), dtype), "values": values, "scale": scale}
    if op == "layer":
        T, E, H, inner = (case[c] for c in "TEHI")
        popularity = 0.5 * torch.randn(E, device=DEVICE, generator=gen)
        logits = torch.randn(T, E, device=DEVICE, generator=gen) + popularity
        up, up_scale = _matrix(gen, (E, H, inner if case["kind"] == "silu" else 2 * inner))
        down, down_scale = _matrix(gen, (E, inner, H))
        most = int(torch.bincount(_choices(logits, case["top_k"])[1].reshape(-1)).max())      # the plain form's rows for each expert
        return {"op": op, "x": _random(gen, (T, H), dtype), "logits": logits, "up": up, "up_scale": up_scale, "down": down,
                "down_scale": down_scale, "top_k": case["top_k"], "kind": case["kind"], "most": most}
    if op == "sort":
        T, E, H = (case[c] for c in "TEH")
        popularity = 0.5 * torch.randn(E, device=DEVICE, generator=gen)
        logits = (torch.randn(T, E, device=DEVICE, generator=gen) + popularity).to(DTYPES[case["logits"]])
        slots = T * case["top_k"]
        return {"op": op, "x": _random(gen, (T, H), dtype).requires_grad_(), "logits": logits.requires_grad_(),
                "y": _random(gen, (slots, H), dtype).requires_grad_(), "grad_sorted": _random(gen, (slots, H), dtype),
                "grad_out": _random(gen, (T, H), dtype), "top_k": case["top_k"], "renormalize": case["renormalize"]}
    if op == "gated":
        columns = case["I"] if case["kind"] == "silu" else 2 * case["I"]
        return {"op": op, "h": _rows(gen, case["rows"], columns, case["pad"], dtype).requires_grad_(),
                "grad": _random(gen, (case["rows"], case["I"]), dtype), "kind": case["kind"]}
    return {"op": op, "x": _rows(gen, case["rows"], case["width"], case["pad"], dtype).requires_grad_(),
            "residual": _random(gen, (case["rows"], case["width"]), dtype) if case["residual"] else None,
            "grad": _random(gen, (case["rows"], case["width"]), dtype), "p": case["p"],
            "rng": torch.randint(0, 1 << 62, (2,), device=DEVICE, generator=gen)}


# ---------------------------------------------------------------------------------------------- one pass
def run(state):
    return {"linear": _run_linear, "layer": _run_layer, "sort": _run_sort, "gated": _run_gated, "dropout": _run_dropout}[state["op"]](state)


def _run_linear(s):
    if own:
        from grouped_mm_bf16_amd import int8
        return int8.linear_int8(s["x"], int8.Columns(s["values"], s["scale"]))
    q, scale = _quantize(s["x"].float())
    return ((q @ s["values"].float()) * scale * s["scale"]).to(s["x"].dtype)


def _quantize(x):
    """Rows as whole numbers of -127 .. 127 (in x's type) and their scales."""
    most = x.abs().amax(-1, keepdim=True).clamp_min(SMALLEST)
    scale = most / torch.full_like(most, 127)
    return torch.round(x / scale), scale


def _choices(logits, top_k):
    """The logits of each token's choices and their experts, the largest first, ties to the lower expert."""
    value, expert = logits.sort(dim=1, descending=True, stable=True)
    return value[:, :top_k], expert[:, :top_k]


def _run_layer(s):
    if own:
        from grouped_mm_bf16_amd import int8
        return int8.moe_forward_int8(s["x"], s["logits"], int8.Columns(s["up"], s["up_scale"]), int8.Columns(s["down"], s["down_scale"]),
                                     s["top_k"], activation=s["kind"])
    return _plain_layer(s)


def _plain_layer(s):
    """Each expert's rows side by side, as many for each as the one with the most has."""
    x, k = s["x"].float(), s["top_k"]
    T, E, most = x.size(0), s["logits"].size(1), s["most"]
    value, expert = _choices(s["logits"].float(), k)
    share = (value - value[:, :1]).exp()
    share = share / share.sum(1, keepdim=True)
    expert = expert.reshape(-1)
    order = torch.argsort(expert, stable=True)
    count = torch.zeros(E, dtype=torch.int64, device=x.device).scatter_add_(0, expert, torch.ones_like(expert))
    place = torch.empty_like(expert)
    place[order] = torch.arange(T * k, device=x.device) - (count.cumsum(0) - count)[expert[order]]
    at = expert * most + place
    q, scale = _quantize(x)
    rows = torch.zeros(E * most, x.size(1), device=x.device)
    rows[at] = q[:, None].expand(T, k, x.size(1)).reshape(T * k, -1)
    h = torch.bmm(rows.reshape(E, most, -1), s["up"].float().contiguous()) * s["up_scale"][:, None]
    h = h.reshape(E * most, -1)[at] * scale[:, None].expand(T, k, 1).reshape(T * k, 1)
    q, scale = _quantize(_activation(h, s["kind"]))
    rows = torch.zeros(E * most, q.size(1), device=x.device)
    rows[at] = q
    y = (torch.bmm(rows.reshape(E, most, -1), s["down"].float().contiguous()) * s["down_scale"][:, None]).reshape(E * most, -1)[at] * scale
    return (y.reshape(T, k, -1) * share[:, :, None]).sum(1).to(s["x"].dtype)


def _activation(h, kind):
    if kind == "silu":
        return h / (1 + (-h).exp())
    inner = h.size(-1) // 2
    return h[:, :inner] / (1 + (-h[:, :inner]).exp()) * h[:, inner:]


def _run_sort(s):
    if own:
        from grouped_mm_bf16_amd import moe_train
        routing = moe_train.route(s["logits"], s["top_k"], s["renormalize"])
        rows = moe_train.sort_rows(s["x"], routing)
        out = moe_train.combine_rows(s["y"], routing, s["top_k"])
        grads = torch.autograd.grad((rows, out), (s["x"], s["y"], s["logits"]), (s["grad_sorted"], s["grad_out"]))
        return {"row_token": routing.row_token, "offs": routing.offs, "sorted": rows.detach(), "out": out.detach(), "grad_x": grads[0],
                "grad_y": grads[1], "grad_logits": grads[2]}
    with torch.no_grad():
        return _plain_sort(s)


def _plain_sort(s):
    x, y, logits, k = s["x"].float(), s["y"].float(), s["logits"].float(), s["top_k"]
    T, E = logits.shape
    value, expert = _choices(logits, k)
    if s["renormalize"]:
        share = (value - value[:, :1]).exp()
        share = share / share.sum(1, keepdim=True)
    else:
        all_shares = (logits - value[:, :1]).exp()
        all_shares = all_shares / all_shares.sum(1, keepdim=True)
        share = all_shares.gather(1, expert)
    slot = torch.argsort(expert.reshape(-1), stable=True)
    token = slot // k
    row = torch.empty_like(slot)
    row[slot] = torch.arange(T * k, device=x.device)
    offs = torch.zeros(E, dtype=torch.int64, device=x.device).scatter_add_(0, expert.reshape(-1), torch.ones_like(slot)).cumsum(0)
    mine = y[row].reshape(T, k, -1)
    grad = s["grad_out"].float()
    grad_share = (mine * grad[:, None]).sum(2)
    if s["renormalize"]:
        grad_logits = torch.zeros_like(logits).scatter_(1, expert, share * (grad_share - (share * grad_share).sum(1, keepdim=True)))
    else:
        grad_logits = torch.zeros_like(logits).scatter_(1, expert, grad_share) - (share * grad_share).sum(1, keepdim=True)
        grad_logits = all_shares * grad_logits
    dtype = s["x"].dtype
    return {"row_token": token.to(torch.int32), "offs": offs.to(torch.int32), "sorted": s["x"][token],
            "out": (mine * share[:, :, None]).sum(1).to(dtype),
            "grad_x": s["grad_sorted"].float()[row].reshape(T, k, -1).sum(1).to(dtype),
            "grad_y": (grad[token] * share.reshape(-1)[slot][:, None]).to(dtype), "grad_logits": grad_logits.to(s["logits"].dtype)}


def _run_gated(s):
    if own:
        from grouped_mm_bf16_amd import moe_train
        out = moe_train.gated(s["h"], s["kind"])
        grad, = torch.autograd.grad(out, s["h"], s["grad"])
        return {"out": out.detach(), "grad_h": grad}
    with torch.no_grad():
        return _plain_gated(s)


def _plain_gated(s):
    h, grad = s["h"].float(), s["grad"].float()
    inner = grad.size(1)
    gate = h[:, :inner]
    part = 1 / (1 + (-gate).exp())
    slope = part * (1 + gate * (1 - part))
    if s["kind"] == "silu":
        out, grad_h = gate * part, grad * slope
    else:
        up = h[:, inner:]
        out, grad_h = gate * part * up, torch.cat([grad * up * slope, grad * gate * part], 1)
    return {"out": out.to(s["h"].dtype), "grad_h": grad_h.to(s["h"].dtype)}


def _run_dropout(s):
    if own:
        from grouped_mm_bf16_amd import dropout
        out = dropout.dropout(s["x"], s["p"], s["rng"], residual=s["residual"])
        grad, = torch.autograd.grad(out, s["x"], s["grad"])
        return {"out": out.detach(), "grad_x": grad}
    with torch.no_grad():
        return _plain_dropout(s)


def _plain_dropout(s):
    x = s["x"].float()
    limit = round(s["p"] * 65536)
    kept = _plain_bits(x.numel(), s["rng"]).reshape(x.shape) >= limit
    factor = 65536 / (65536 - limit)
    out = torch.where(kept, x * factor, 0.0)
    if s["residual"] is not None:
        out = s["residual"].float() + out
    return {"out": out.to(s["x"].dtype), "grad_x": torch.where(kept, s["grad"].float() * factor, 0.0).to(s["x"].dtype)}


def _plain_bits(n, rng):
    """16 random bits for each of n elements: eight to a block of Philox 4x32-10 (Salmon, Moraes, Dror, Shaw 2011), whose key is rng[0] and
    whose counter is the block's number and rng[1]; a word's lower half first.  64-bit products wrap, their bits 0 to 63 are right."""
    low = 0xffffffff
    block = torch.arange((n + 7) // 8, device=rng.device)
    seed, offset = rng[0], rng[1]
    k0, k1 = seed & low, seed >> 32 & low
    c0, c1, c2, c3 = block & low, block >> 32, (offset & low).expand_as(block), (offset >> 32 & low).expand_as(block)
    for _ in range(10):
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = (p1 >> 32 & low) ^ c1 ^ k0, p1 & low, (p0 >> 32 & low) ^ c3 ^ k1, p0 & low
        k0, k1 = k0 + 0x9E3779B9 & low, k1 + 0xBB67AE85 & low
    words = torch.stack([c0, c1, c2, c3], 1)
    return torch.stack([words & 0xffff, words >> 16], 2).reshape(-1)[:n]


# ---------------------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    s = {name: t.detach() if torch.is_tensor(t) else t for name, t in prepare(case, seed).items()}
    return {"linear": _exact_linear, "layer": _exact_layer, "sort": _exact_sort, "gated": _exact_gated, "dropout": _exact_dropout}[case["op"]](s)


def _steps(x):
    """Rows rounded to whole steps of a 127th of their largest element, times that step."""
    step = torch.clamp(x.abs().max(dim=1, keepdim=True).values, min=SMALLEST) / 127
    return torch.round(x / step) * step


def _exact_linear(s):
    return _steps(s["x"].double()) @ (s["values"].double() * s["scale"].double())


def _exact_layer(s):
    """Expert by expert, on the tokens that chose it."""
    x, k = _steps(s["x"].double()), s["top_k"]
    order = torch.argsort(s["logits"].double(), dim=1, descending=True, stable=True)[:, :k]
    weight = torch.softmax(s["logits"].double().gather(1, order), dim=1)
    out = torch.zeros_like(x)
    for e in order.unique().tolist():
        token, choice = (order == e).nonzero(as_tuple=True)
        h = (x[token] @ s["up"][e].double()) * s["up_scale"][e].double()
        if s["kind"] == "silu":
            a = torch.sigmoid(h) * h
        else:
            gate, up = h.chunk(2, dim=1)
            a = torch.sigmoid(gate) * gate * up
        y = (_steps(a) @ s["down"][e].double()) * s["down_scale"][e].double()
        out.index_add_(0, token, y * weight[token, choice][:, None])
    return out


def _exact_sort(s):
    """Token by token's choices as a sparse matrix of weights between tokens and rows."""
    logits, k = s["logits"].double(), s["top_k"]
    T, E = logits.shape
    chosen = torch.argsort(logits, dim=1, descending=True, stable=True)[:, :k]
    among = torch.full_like(logits, -math.inf).scatter(1, chosen, logits.gather(1, chosen)) if s["renormalize"] else logits
    share = torch.softmax(among, dim=1)
    # rows in the order of (expert, token, choice): the number of a slot's expert, then the slot's own
    rank = torch.argsort(chosen.reshape(-1) * (T * k) + torch.arange(T * k, device=logits.device))
    token = torch.div(rank, k, rounding_mode="floor")
    expert = chosen.reshape(-1)[rank]
    x, y, back, grad = s["x"].double(), s["y"].double(), s["grad_sorted"].double(), s["grad_out"].double()
    weight = share[token, expert][:, None]
    grad_x = torch.zeros_like(x).index_add_(0, token, back)
    out = torch.zeros_like(x).index_add_(0, token, y * weight)
    grad_share = torch.zeros_like(share)
    grad_share[token, expert] = torch.linalg.vecdot(y, grad[token])
    # softmax's own derivative, over what it was taken over
    grad_logits = share * grad_share - share * torch.linalg.vecdot(share, grad_share)[:, None]
    return {"row_token": token.to(torch.int32), "offs": torch.bincount(expert, minlength=E).cumsum(0).to(torch.int32), "sorted": x[token],
            "out": out, "grad_x": grad_x, "grad_y": grad[token] * weight, "grad_logits": grad_logits}


def _exact_gated(s):
    with torch.enable_grad():
        h = s["h"].double().requires_grad_()
        out = torch.nn.functional.silu(h) if s["kind"] == "silu" else torch.nn.functional.silu(h[:, :h.size(1) // 2]) * h[:, h.size(1) // 2:]
        grad, = torch.autograd.grad(out, h, s["grad"].double())
    return {"out": out.detach(), "grad_h": grad}


def _exact_dropout(s):
    """The random bits on the host, in unsigned 64-bit numbers."""
    x, (seed, offset) = s["x"].double(), (v & 0xffffffffffffffff for v in s["rng"].tolist())
    n = x.numel()
    low, half = np.uint64(0xffffffff), np.uint64(32)
    number = np.arange(-(-n // 8), dtype=np.uint64)
    counter = [number & low, number >> half, np.full_like(number, offset & 0xffffffff), np.full_like(number, offset >> 32)]
    for turn in range(10):
        key = [np.uint64((seed & 0xffffffff) + turn * 0x9E3779B9 & 0xffffffff), np.uint64((seed >> 32) + turn * 0xBB67AE85 & 0xffffffff)]
        a, b = counter[0] * np.uint64(0xD2511F53), counter[2] * np.uint64(0xCD9E8D57)
        counter = [b >> half ^ counter[1] ^ key[0], b & low, a >> half ^ counter[3] ^ key[1], a & low]
    bits = np.stack(counter, 1).astype("<u4").view("<u2").reshape(-1)[:n]
    kept = torch.from_numpy((bits >= round(s["p"] * 65536)).reshape(x.shape)).to(x.device).double()
    factor = kept / (1 - round(s["p"] * 65536) / 65536)
    out = x * factor
    return {"out": out if s["residual"] is None else out + s["residual"].double(), "grad_x": s["grad"].double() * factor}


# ---------------------------------------------------------------------------------------------- what it takes
def work(case):
    size = BYTES[case["dtype"]]
    if case["op"] == "linear":
        T, K, N = (case[c] for c in "TKN")
        return {"bytes": size * T * (K + N) + K * N + 4 * N, "flops": 2 * T * K * N}
    if case["op"] == "layer":
        T, E, k, H, inner = (case[c] for c in ("T", "E", "top_k", "H", "I"))
        touched = E * (1.0 - (1.0 - k / E) ** T)                    # experts that at least one token chooses
        return {"bytes": int(size * 2 * T * H + 4 * T * E + touched * (_weights(case) + 4 * (_weights(case) // H - inner + H))),
                "flops": 2 * T * k * _weights(case)}
    if case["op"] == "sort":
        T, E, k, H = (case[c] for c in ("T", "E", "top_k", "H"))
        # x, y and both gradients in; rows, result and both gradients out; the logits and their gradient; row numbers
        return {"bytes": size * T * H * (4 + 4 * k) + 2 * T * E * BYTES[case["logits"]] + 4 * (T * k + E), "flops": 6 * T * k * H}
    if case["op"] == "gated":
        elements, parts = case["rows"] * case["I"], 1 if case["kind"] == "silu" else 2
        return {"bytes": size * elements * (2 + 2 * parts), "flops": 20 * elements}
    elements = case["rows"] * case["width"]
    return {"bytes": size * elements * (4 + (1 if case["residual"] else 0)), "flops": 4 * elements}
