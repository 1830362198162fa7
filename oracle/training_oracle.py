"""64-bit restatements of the operators around the grouped products of an expert layer that is trained, and of dropout, on the CPU, from their
formulas, with bounds of what fp32 arithmetic and one rounding leave.  Used by the tests only; independent of the package."""
import numpy as np
import torch

from .operators_oracle import EPS32, TINY, UNIT, f64

SMALLEST32 = 2.0 ** -126     # of a normal fp32 value


def _slots(token_rows, tokens):
    return token_rows.cpu().long().reshape(tokens, -1)


def sorted_rows(x, token_rows):
    """Row token_rows[t, j] = x[t], bit for bit."""
    at = _slots(token_rows, x.size(0))
    out = torch.empty(at.numel(), x.size(1), dtype=x.dtype)
    for j in range(at.size(1)):
        out[at[:, j]] = x.detach().cpu()
    return out


def sum_rows(y, token_rows, weight, tokens):
    """sum over j of weight[t, j] y[token_rows[t, j]], and its bound: one rounding, a product and a sum in fp32 for each term."""
    at = _slots(token_rows, tokens)
    terms = f64(y)[at]
    if weight is not None:
        terms = terms * f64(weight).reshape(tokens, -1, 1)
    out = terms.sum(1)
    return out, UNIT[y.dtype] * out.abs() + TINY[y.dtype] + (at.size(1) + 1) * EPS32 * terms.abs().sum(1)


def combine_backward(grad, y, token_rows, weight):
    """dy and its bound, dweight and its bound (sums of at most width / 64 + 8 terms one after the other, then a tree of 64)."""
    tokens = grad.size(0)
    at, d, w = _slots(token_rows, tokens), f64(grad), f64(weight).reshape(tokens, -1)
    dy = torch.zeros(at.numel(), grad.size(1), dtype=torch.float64)
    dy[at.reshape(-1)] = (d[:, None] * w[:, :, None]).reshape(at.numel(), -1)
    terms = f64(y)[at] * d[:, None]
    return (dy, UNIT[grad.dtype] * dy.abs() + TINY[grad.dtype] + EPS32 * dy.abs(),
            terms.sum(2).reshape(-1), ((grad.size(1) / 64 + 16) * EPS32 * terms.abs().sum(2)).reshape(-1) + 2.0 ** -149 * grad.size(1))


def route_backward(grad, slot_expert, slot_weight, logits, renormalize):
    """dlogits and its bound, for the weights as they were written."""
    tokens, experts = logits.shape
    chosen, w, g = slot_expert.cpu().long().reshape(tokens, -1), f64(slot_weight).reshape(tokens, -1), f64(grad).reshape(tokens, -1)
    s, size = (w * g).sum(1, keepdim=True), (w * g).abs().sum(1, keepdim=True)
    if renormalize:
        p, off = torch.zeros(tokens, experts, dtype=torch.float64), torch.zeros(tokens, experts, dtype=torch.float64)
    else:
        z = f64(logits)
        best = z.max(1, keepdim=True).values
        down = torch.where(z == best, torch.zeros_like(z), z - best)
        p = torch.exp(down)
        p = p / p.sum(1, keepdim=True)
        off = (32 + down.abs().nan_to_num(posinf=0)) * EPS32 * p
    p = p.scatter(1, chosen, w)
    off = off.scatter(1, chosen, torch.zeros_like(w))
    d = torch.zeros(tokens, experts, dtype=torch.float64).scatter(1, chosen, g)
    out = p * (d - s)
    return out, UNIT[logits.dtype] * out.abs() + TINY[logits.dtype] + p * EPS32 * (3 * (d.abs() + s.abs()) + 10 * size) + off * (d.abs() + size)


def gated(h, kind):
    """The activation and its bound: e^-g to a few units of fp32 and as many as the exponent's rounding leaves, then six roundings."""
    h64, dtype = f64(h), h.dtype
    inner = h.size(1) // (2 if kind == "swiglu" else 1)
    g, u = h64[:, :inner], h64[:, inner:] if kind == "swiglu" else torch.ones(h.size(0), inner, dtype=torch.float64)
    out = g * torch.sigmoid(g) * u
    return out, UNIT[dtype] * out.abs() + TINY[dtype] + (10 + 2 * g.abs()) * EPS32 * out.abs() + 2 * SMALLEST32 * (g * u).abs()


def gated_backward(grad, h, kind):
    h64, d, dtype = f64(h), f64(grad), h.dtype
    inner = grad.size(1)
    g = h64[:, :inner]
    part, rest = torch.sigmoid(g), torch.sigmoid(-g)
    size = d.abs() * part * (1 + g.abs() * rest)
    rough = (16 + 2 * g.abs()) * EPS32
    low = 2 * SMALLEST32 * d.abs() * (1 + g.abs())
    dg = d * part * (1 + g * rest)
    if kind == "silu":
        return dg, UNIT[dtype] * dg.abs() + TINY[dtype] + rough * size + low
    u = h64[:, inner:]
    du = d * g * part
    dg = dg * u
    out = torch.cat([dg, du], 1)
    bound = torch.cat([rough * size * u.abs() + low * u.abs(), rough * du.abs() + low], 1)
    return out, UNIT[dtype] * out.abs() + TINY[dtype] + bound


def dropout_bits(n, seed, offset, site=0, first=0):
    """16 bits for each of n elements from element 8 * first on, from Philox 4x32-10 in Python's own whole numbers, a block at a time."""
    low, blocks = 0xffffffff, []
    for b in range(first, first - (-n // 8)):
        c = [b & low, (b >> 32 | site << 16) & low, offset & low, offset >> 32 & low]
        k = [seed & low, seed >> 32 & low]
        for _ in range(10):
            p, q = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
            c = [q >> 32 ^ c[1] ^ k[0], q & low, p >> 32 ^ c[3] ^ k[1], p & low]
            k = [k[0] + 0x9E3779B9 & low, k[1] + 0xBB67AE85 & low]
        blocks += [v >> s & 0xffff for v in c for s in (0, 16)]
    return np.array(blocks[:n], dtype=np.int64)


def dropout(x, p, seed, offset, site=0, residual=None):
    """The result, its bound, and what was kept."""
    limit = round(p * 65536)
    kept = torch.from_numpy(dropout_bits(x.numel(), seed, offset, site) >= limit).reshape(x.shape)
    x64 = torch.where(kept, f64(x), torch.zeros((), dtype=torch.float64))
    out = x64 * (65536 / (65536 - limit)) if limit < 65536 else torch.zeros_like(x64)
    size = 2 * out.abs()
    if residual is not None:
        out = out + f64(residual)
        size = size + f64(residual).abs()
    return out, UNIT[x.dtype] * out.abs() + TINY[x.dtype] + 2 * EPS32 * size, kept
