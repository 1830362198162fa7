"""Operators around the grouped product, as measurable cases: a shared projection with the low-rank adapters of many requests
(``lora.lora_linear``), the whole mixture-of-experts layer for a few tokens (``moe.moe_forward_few``), layer norm (``norm.layer_norm``).

``own`` false: the operators in their plain form, elementary torch operations in 32 bits, rounded once at the end.  ``own`` true: the
calls that a user of the package makes.  Ranges that the listed cases stand for:

    adapters       1 to 8192 tokens of 1 to 256 requests, 1 to 64 adapters of rank 1 to 128 (and tokens without one), inner and outer
                   size 64 to 8192; bf16 and fp16; weights and adapters row-major or as linear layers store them; sizes without any
                   alignment; forward, and a training step of the adapters beside a frozen projection
    expert layers  1 to 64 tokens, 4 to 128 experts, 1 to 8 choices, hidden size 256 to 4096, inner size 128 to 14336, weights up to
                   3 GB; bf16 and fp16; SwiGLU with gate and up columns apart or interleaved, SiLU; row- or column-major weights
    layer norm     1 to 65536 rows of 64 to 16384 elements; bf16, fp16, fp32; rows that lie apart; forward, and forward with backward
"""
from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
MAX_LORA_FLOPS = 7e11      # a drawn case costs no more than the largest listed one
MAX_LAYER_BYTES = 3.0e9
MAX_NORM_ELEMENTS = 1.4e8


# ---------------------------------------------------------------------------------------------- cases
def _lora(tokens, requests, adapters, rank, inner, outer, dtype="bf16", linear=False, pad=0, train=False):
    """linear: the projection and the adapters lie as linear layers store them ([out, in]).  pad: x is a slice of rows that much longer."""
    return {"op": "lora", "T": tokens, "requests": requests, "L": adapters, "R": rank, "K": inner, "N": outer, "dtype": dtype,
            "linear": linear, "pad": pad, "train": train}


def _layer(tokens, experts, top_k, hidden, inner, kind="swiglu", col=False, dtype="bf16", logits="fp32"):
    return {"op": "layer", "T": tokens, "E": experts, "top_k": top_k, "H": hidden, "I": inner, "kind": kind, "col": col,
            "dtype": dtype, "logits": logits}


def _norm(rows, width, dtype="bf16", pad=0, train=False):
    return {"op": "norm", "rows": rows, "width": width, "dtype": dtype, "pad": pad, "train": train}


def listed():
    cases = {
        # one sequence is being answered, with its adapter: the output projection of a block, latency alone
        "lora_one": _lora(1, 1, 8, 16, 4096, 4096),
        # a decoding step of 48 sequences, each with an adapter of its own choice, through a wide projection stored as a linear layer
        "lora_decode": _lora(48, 48, 64, 16, 4096, 8192, linear=True),
        # the prompts of six requests in one batch, x a part of a wider buffer
        "lora_prefill": _lora(4096, 6, 16, 64, 4096, 4096, pad=4096),
        # a training step of eight adapters at once, one sequence each, beside a frozen projection
        "lora_train": _lora(8192, 8, 8, 16, 4096, 4096, train=True),
        # a training step whose sizes have no alignment at all, half precision
        "lora_odd_train": _lora(615, 5, 3, 5, 1031, 519, dtype="fp16", train=True),
        # one token through many small experts: latency
        "few_one_small": _layer(1, 128, 8, 2048, 768),
        # eight sequences through few large experts whose weights were prepared for the fused activation
        "few_large": _layer(8, 8, 2, 4096, 14336, kind="interleaved"),
        # 32 sequences through many small experts stored as linear layers, half precision
        "few_batch_small": _layer(32, 128, 8, 2048, 768, col=True, dtype="fp16", logits="fp16"),
        # a decoding step's norm: latency alone
        "norm_decode": _norm(32, 4096),
        # the norm of a training step, both directions
        "norm_train": _norm(16384, 4096, train=True),
        # full precision, odd width, rows apart, both directions
        "norm_odd_train": _norm(3001, 1031, dtype="fp32", pad=5, train=True),
        # a long prompt through a wide norm, half precision
        "norm_prefill": _norm(8192, 14336, dtype="fp16"),
    }
    return [dict(case, name=name) for name, case in cases.items()]


def _log(rng, lo, hi):
    """Whole number between lo and hi, uniform in its logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _draw_lora(rng):
    odd, train = rng.random() < 0.25, rng.random() < 0.4
    tokens = _log(rng, 16 if train else 1, 8192)
    if not train and rng.random() < 0.4:
        tokens = _log(rng, 1, 256)
        requests = tokens                      # a decoding step
    else:
        requests = min(tokens, _log(rng, 1, 32))
    inner, outer = _log(rng, 64, 8192), _log(rng, 64, 8192)
    rank = rng.choice([_log(rng, 1, 128), 8, 16, 32, 64])
    if not odd:
        inner, outer = inner // 8 * 8, outer // 8 * 8
    pad = rng.choice([0, 0, inner, 24]) + (rng.randrange(8) if odd else 0)
    return _lora(tokens, requests, _log(rng, 1, 64), rank, inner, outer, dtype=rng.choice(["bf16", "bf16", "fp16"]),
                 linear=rng.random() < 0.5, pad=pad, train=train)


def _draw_layer(rng):
    kind = rng.choice(["swiglu", "swiglu", "interleaved", "silu"])
    experts = _log(rng, 4, 128)
    hidden, inner = _log(rng, 256, 4096), _log(rng, 128, 14336)
    if kind == "interleaved":
        inner = inner // 64 * 64
    elif rng.random() < 0.8:
        inner = inner // 8 * 8
    if rng.random() < 0.85:
        hidden = hidden // 8 * 8
    return _layer(_log(rng, 1, 64), experts, rng.randint(1, min(8, experts)), hidden, inner, kind=kind, col=rng.random() < 0.35,
                  dtype=rng.choice(["bf16", "bf16", "fp16"]), logits=rng.choice(["fp32", "fp32", "bf16", "fp16"]))


def _draw_norm(rng):
    return _norm(_log(rng, 1, 65536), _log(rng, 64, 16384), dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                 pad=rng.choice([0, 0, 8, 3]), train=rng.random() < 0.6)


def draw(rng):
    while True:
        case = rng.choice([_draw_lora, _draw_layer, _draw_norm])(rng)
        if case["op"] == "lora" and work(case)["flops"] <= MAX_LORA_FLOPS:
            return case
        if case["op"] == "layer" and _weights(case) * case["E"] * BYTES[case["dtype"]] <= MAX_LAYER_BYTES:
            return case
        if case["op"] == "norm" and case["rows"] * case["width"] <= MAX_NORM_ELEMENTS * (0.5 if case["train"] else 1.0):
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


def _adapters_of(case, seed):
    """Adapter of each token: the requests follow one another and hold at least one token each; about one in eight has no adapter."""
    T, n, L = case["T"], case["requests"], case["L"]
    gen = torch.Generator().manual_seed(seed)
    cuts = (torch.randperm(T - 1, generator=gen)[:n - 1] + 1).sort().values
    request = torch.zeros(T, dtype=torch.int64)
    request[cuts] = 1
    request = request.cumsum(0)
    which = torch.randint(0, L, (n,), generator=gen)
    if n > 2:
        which = torch.where(torch.rand(n, generator=gen) < 0.125, torch.full_like(which, -1), which)
    return which[request].to(torch.int32).to(DEVICE)


def _matrix(gen, shape, dtype, scale, turned):
    """A (stack of) matrices of this shape; turned: the last two dimensions are swapped in memory."""
    if not turned:
        return _random(gen, shape, dtype, scale)
    return _random(gen, shape[:-2] + (shape[-1], shape[-2]), dtype, scale).transpose(-2, -1)


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    if case["op"] == "lora":
        T, L, R, K, N = (case[c] for c in "TLRKN")
        state = {"op": "lora", "train": case["train"], "x": _rows(gen, T, K, case["pad"], dtype),
                 "weight": _matrix(gen, (K, N), dtype, K ** -0.5, case["linear"]),
                 "lora_a": _matrix(gen, (L, K, R), dtype, K ** -0.5, case["linear"]),
                 "lora_b": _matrix(gen, (L, R, N), dtype, R ** -0.5, case["linear"]),
                 "adapter": _adapters_of(case, seed), "scale": 0.25 + 0.75 * torch.rand(L, device=DEVICE, generator=gen)}
        if case["train"]:
            for name in ("x", "lora_a", "lora_b"):
                state[name] = state[name].detach().requires_grad_()
            state["grad"] = _random(gen, (T, N), dtype)
        return state
    if case["op"] == "layer":
        T, E, H, inner, kind = case["T"], case["E"], case["H"], case["I"], case["kind"]
        popularity = 0.5 * torch.randn(E, device=DEVICE, generator=gen)
        logits = torch.randn(T, E, device=DEVICE, generator=gen) + popularity
        # "interleaved": 64 gate columns, then their 64 partners, and so on
        return {"op": "layer", "x": _random(gen, (T, H), dtype), "logits": logits.to(DTYPES[case["logits"]]),
                "w_up": _matrix(gen, (E, H, inner if kind == "silu" else 2 * inner), dtype, H ** -0.5, case["col"]),
                "w_down": _matrix(gen, (E, inner, H), dtype, inner ** -0.5, case["col"]), "top_k": case["top_k"], "kind": kind}
    rows, width = case["rows"], case["width"]
    state = {"op": "norm", "train": case["train"], "x": _rows(gen, rows, width, case["pad"], dtype).mul_(2.0).add_(0.5),
             "weight": _random(gen, (width,), dtype, 0.2).add_(1.0), "bias": _random(gen, (width,), dtype, 0.2), "eps": 1e-5}
    if case["train"]:
        for name in ("x", "weight", "bias"):
            state[name] = state[name].detach().requires_grad_()
        state["grad"] = _random(gen, (rows, width), dtype)
    return state


# ---------------------------------------------------------------------------------------------- one pass
def run(state):
    return {"lora": _run_lora, "layer": _run_layer, "norm": _run_norm}[state["op"]](state)


def _run_lora(s):
    if own:
        from grouped_mm_bf16_amd import lora
        out = lora.lora_linear(s["x"], s["weight"], s["lora_a"], s["lora_b"], s["adapter"], s["scale"])
        if not s["train"]:
            return out
        grads = torch.autograd.grad(out, (s["x"], s["lora_a"], s["lora_b"]), s["grad"])
        return {"out": out.detach(), "grad_x": grads[0], "grad_a": grads[1], "grad_b": grads[2]}
    with torch.no_grad():
        return _plain_lora(s)


def _plain_lora(s):
    """All adapters' products of all tokens, those of other adapters set to zero in between."""
    x, weight = s["x"].float(), s["weight"].float()
    L, K, R = s["lora_a"].shape
    a = s["lora_a"].float().permute(1, 0, 2).reshape(K, L * R)
    b = s["lora_b"].float().reshape(L * R, -1)
    mine = (s["adapter"][:, None] == torch.arange(L, device=x.device)).float() * s["scale"]
    mine = mine[:, :, None].expand(-1, -1, R).reshape(-1, L * R)
    v = (x @ a) * mine
    out = (x @ weight + v @ b).to(s["x"].dtype)
    if not s["train"]:
        return out
    grad = s["grad"].float()
    u = (grad @ b.t()) * mine
    grad_x = grad @ weight.t() + u @ a.t()
    grad_a = (x.t() @ u).reshape(K, L, R).permute(1, 0, 2)
    grad_b = (v.t() @ grad).reshape(L, R, -1)
    return {"out": out, "grad_x": grad_x.to(out.dtype), "grad_a": grad_a.to(out.dtype), "grad_b": grad_b.to(out.dtype)}


def _run_layer(s):
    if own:
        from grouped_mm_bf16_amd import moe
        return moe.moe_forward_few(s["x"], s["logits"], s["w_up"], s["w_down"], s["top_k"],
                                   activation="silu" if s["kind"] == "silu" else "swiglu", interleaved=s["kind"] == "interleaved")
    return _plain_layer(s)


def _plain_layer(s):
    """Each slot's own copy of its expert's weights where that is fewer than the experts, else every token through all of them."""
    x, k = s["x"].float(), s["top_k"]
    T, E = s["logits"].shape
    value, expert = s["logits"].float().sort(dim=1, descending=True, stable=True)
    value, expert = value[:, :k], expert[:, :k]
    share = (value - value[:, :1]).exp()
    share = share / share.sum(1, keepdim=True)
    if T * k < E:
        rows = x[:, None].expand(T, k, x.size(1)).reshape(T * k, 1, x.size(1))
        picked = expert.reshape(-1)
        h = _plain_activation(torch.bmm(rows, s["w_up"][picked].float().contiguous()), s["kind"])
        y = torch.bmm(h, s["w_down"][picked].float().contiguous()).reshape(T, k, -1)
        return (y * share[:, :, None]).sum(1).to(s["x"].dtype)
    weight = torch.zeros(T, E, device=x.device).scatter_(1, expert, share)
    h = _plain_activation(torch.matmul(x, s["w_up"].float().contiguous()), s["kind"])
    y = torch.bmm(h, s["w_down"].float().contiguous())
    return (y * weight.t()[:, :, None]).sum(0).to(s["x"].dtype)


def _plain_activation(h, kind):
    if kind == "silu":
        return h / (1 + (-h).exp())
    inner = h.size(-1) // 2
    if kind == "interleaved":
        h = h.reshape(h.shape[:-1] + (inner // 64, 2, 64))
        gate, up = h[..., 0, :].flatten(-2), h[..., 1, :].flatten(-2)
    else:
        gate, up = h[..., :inner], h[..., inner:]
    return gate / (1 + (-gate).exp()) * up


def _run_norm(s):
    if own:
        from grouped_mm_bf16_amd import norm
        out = norm.layer_norm(s["x"], s["weight"], s["bias"], s["eps"])
        if not s["train"]:
            return out
        grads = torch.autograd.grad(out, (s["x"], s["weight"], s["bias"]), s["grad"])
        return {"out": out.detach(), "grad_x": grads[0], "grad_weight": grads[1], "grad_bias": grads[2]}
    with torch.no_grad():
        return _plain_norm(s)


def _plain_norm(s):
    x, weight = s["x"].float(), s["weight"].float()
    centred = x - x.mean(1, keepdim=True)
    rstd = ((centred * centred).mean(1, keepdim=True) + s["eps"]).rsqrt()
    hat = centred * rstd
    out = (hat * weight + s["bias"].float()).to(s["x"].dtype)
    if not s["train"]:
        return out
    grad = s["grad"].float()
    g = grad * weight
    grad_x = rstd * (g - g.mean(1, keepdim=True) - hat * (g * hat).mean(1, keepdim=True))
    return {"out": out, "grad_x": grad_x.to(out.dtype), "grad_weight": (grad * hat).sum(0).to(out.dtype),
            "grad_bias": grad.sum(0).to(out.dtype)}


# ---------------------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    s = {name: t.detach() if torch.is_tensor(t) else t for name, t in prepare(case, seed).items()}
    if case["op"] == "lora":
        return _exact_lora(s)
    return _exact_layer(s) if case["op"] == "layer" else _exact_norm(s)


def _exact_lora(s):
    """Adapter by adapter, on the tokens that it has."""
    x, weight = s["x"].double(), s["weight"].double()
    out = x @ weight
    grads = None
    if s["train"]:
        dy = s["grad"].double()
        grads = [dy @ weight.T, torch.zeros(s["lora_a"].shape, dtype=torch.float64, device=x.device),
                 torch.zeros(s["lora_b"].shape, dtype=torch.float64, device=x.device)]
    for i in s["adapter"].unique().tolist():
        if i < 0:
            continue
        at = (s["adapter"] == i).nonzero()[:, 0]
        a, b, alpha = s["lora_a"][i].double(), s["lora_b"][i].double(), s["scale"][i].double()
        low = x[at] @ a
        out[at] += alpha * (low @ b)
        if grads:
            back = alpha * (dy[at] @ b.T)
            grads[0][at] += back @ a.T
            grads[1][i] = x[at].T @ back
            grads[2][i] = alpha * (low.T @ dy[at])
    if not grads:
        return out
    return {"out": out, "grad_x": grads[0], "grad_a": grads[1], "grad_b": grads[2]}


def _exact_layer(s):
    """Expert by expert, on the tokens that chose it."""
    x, logits, k = s["x"].double(), s["logits"].double(), s["top_k"]
    order = torch.argsort(logits, dim=1, descending=True, stable=True)[:, :k]
    weight = torch.softmax(logits.gather(1, order), dim=1)
    out = torch.zeros_like(x)
    for e in order.unique().tolist():
        token, choice = (order == e).nonzero(as_tuple=True)
        h = x[token] @ s["w_up"][e].double()
        if s["kind"] == "silu":
            h = h * torch.sigmoid(h)
        else:
            half = h.size(1) // 2
            column = torch.arange(half, device=x.device)
            gate = column if s["kind"] == "swiglu" else column // 64 * 128 + column % 64
            g, u = h[:, gate], h[:, gate + (half if s["kind"] == "swiglu" else 64)]
            h = g * torch.sigmoid(g) * u
        out.index_add_(0, token, (h @ s["w_down"][e].double()) * weight[token, choice][:, None])
    return out


def _exact_norm(s):
    x, w = s["x"].double(), s["weight"].double()
    var, mean = torch.var_mean(x, dim=1, correction=0, keepdim=True)
    z = (x - mean) / torch.sqrt(var + s["eps"])
    out = z * w + s["bias"].double()
    if not s["train"]:
        return out
    dy = s["grad"].double()
    dz = dy * w
    n = x.size(1)
    dx = (n * dz - dz.sum(1, keepdim=True) - z * (dz * z).sum(1, keepdim=True)) / (n * torch.sqrt(var + s["eps"]))
    return {"out": out, "grad_x": dx, "grad_weight": (dy * z).sum(0), "grad_bias": dy.sum(0)}


# ---------------------------------------------------------------------------------------------- what it takes
def work(case):
    size = BYTES[case["dtype"]]
    if case["op"] == "lora":
        T, L, R, K, N = (case[c] for c in "TLRKN")
        used = L * (1.0 - (1.0 - 1.0 / L) ** case["requests"])      # adapters that at least one request has
        low = used * R * (K + N)
        moved = T * (K + N) + K * N + low
        flops = 2 * T * K * N + 2 * T * R * (K + N)
        if case["train"]:      # the output's gradient in; x's and all adapters' gradients out
            moved += T * (K + N) + L * R * (K + N)
            flops = 4 * T * K * N + 6 * T * R * (K + N)
        return {"bytes": int(moved * size + 4 * T), "flops": int(flops)}
    if case["op"] == "layer":
        T, E, k, H = case["T"], case["E"], case["top_k"], case["H"]
        touched = E * (1.0 - (1.0 - k / E) ** T)                    # experts that at least one token chooses
        return {"bytes": int(size * (2 * T * H + touched * _weights(case)) + T * E * BYTES[case["logits"]]),
                "flops": 2 * T * k * _weights(case)}
    elements = case["rows"] * case["width"]
    if not case["train"]:
        return {"bytes": int(size * (2 * elements + 2 * case["width"])), "flops": 8 * elements}
    return {"bytes": int(size * (4 * elements + 4 * case["width"])), "flops": 20 * elements}
