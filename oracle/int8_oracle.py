"""Restatement of the 8-bit products on the CPU: rounding in the same fp32 operations, everything behind it in 64 bits.  Used by the tests only;
independent of the package."""
import torch

from .operators_oracle import EPS32, TINY, UNIT, f64


def quantize(x):
    """Whole numbers (float64) and float32 scales of the rows: fp32's division and its rounding to even are exact by definition."""
    x = x.detach().cpu().float()
    most = x.abs().amax(1) if x.size(1) else torch.zeros(x.size(0))
    most = torch.where(most < 2.0 ** -100, torch.full_like(most, 2.0 ** -100), most)
    most = torch.where(x.isnan().any(1), torch.full_like(most, float("nan")), most) if x.size(1) else most
    scale = most / torch.full_like(most, 127)
    q = torch.round(x / scale[:, None])
    return torch.where(torch.isfinite(most)[:, None], q, torch.zeros_like(q)).double(), scale


def mm(a, a_scale, b, b_scale, dtype):
    """(a * a_scale) @ (b * b_scale) and its bound: the sum's rounding to fp32, two products, the result's rounding.  a [M, K], b [K, N]."""
    total = a.cpu().double() @ b.cpu().double()
    out = total * f64(a_scale)[:, None] * f64(b_scale)[None]
    return out, UNIT[dtype] * out.abs() + TINY[dtype] + 4 * EPS32 * out.abs()


def grouped_mm(a, a_scale, b, b_scale, offs, dtype, row_index=None):
    """The same of jagged rows, and which rows a group has."""
    if row_index is not None:
        index = row_index.cpu().long()
        there = (index >= 0) & (index < a.size(0))
        a = torch.where(there[:, None], a.cpu()[index.clamp(0, a.size(0) - 1)], torch.zeros((), dtype=a.dtype))
        a_scale = torch.where(there, a_scale.cpu()[index.clamp(0, a_scale.numel() - 1)], torch.zeros(()))
    M, N = a.size(0), b.size(2)
    out, bound, owned = torch.zeros(M, N, dtype=torch.float64), torch.zeros(M, N, dtype=torch.float64), torch.zeros(M, dtype=torch.bool)
    first = 0
    for g, end in enumerate(offs.tolist()):
        if end > first:
            out[first:end], bound[first:end] = mm(a[first:end], a_scale[first:end], b[g], b_scale[g], dtype)
            owned[first:end] = True
        first = max(first, end)
    return out, bound, owned


def layer(x, logits, up, up_scale, down, down_scale, top_k, kind, renormalize=True):
    """The expert layer in 64 bits, its activations rounded to 8 bits where the kernels do, and in the same steps."""
    x8, x_scale = quantize(x)
    z = f64(logits)
    chosen = torch.argsort(z, dim=1, descending=True, stable=True)[:, :top_k]
    weight = torch.softmax(z.gather(1, chosen), 1) if renormalize else torch.softmax(z, 1).gather(1, chosen)
    out = torch.zeros(x.shape, dtype=torch.float64)
    for e in chosen.unique().tolist():
        token, j = (chosen == e).nonzero(as_tuple=True)
        h = (x8[token] @ up[e].cpu().double()) * f64(x_scale)[token, None] * f64(up_scale[e])
        inner = down.size(1)
        a = torch.nn.functional.silu(h) if kind == "silu" else torch.nn.functional.silu(h[:, :inner]) * h[:, inner:]
        a8, a_scale = quantize(a)
        y = (a8 @ down[e].cpu().double()) * f64(a_scale)[:, None] * f64(down_scale[e])
        out.index_add_(0, token, y * weight[token, j][:, None])
    return out


def layer_within(x, logits, up, up_scale, down, down_scale, top_k, kind, renormalize=True):
    """:func:`layer` and its bound element by element.

    The activation in fp32: the sums are exact, three roundings make a gate (and its partner) of them, e^-g takes a few units and as many as its
    argument's rounding leaves, then three roundings.  What that leaves decides a value's step of 8 bits only where the quotient lies that near a half:
    those values may be a whole step off, the others are none, and a row's scale is off as its largest value is.  The experts' rows and their sum stay in
    fp32, one rounding follows."""
    dtype = x.dtype
    x8, x_scale = quantize(x)
    z = f64(logits)
    chosen = torch.argsort(z, dim=1, descending=True, stable=True)[:, :top_k]
    weight = torch.softmax(z.gather(1, chosen), 1) if renormalize else torch.softmax(z, 1).gather(1, chosen)
    weight_err = (16 + 4 * (z.max(1).values - z.min(1).values))[:, None] * EPS32 * weight
    out, bound = torch.zeros(x.shape, dtype=torch.float64), torch.zeros(x.shape, dtype=torch.float64)
    inner = down.size(1)
    for e in chosen.unique().tolist():
        token, j = (chosen == e).nonzero(as_tuple=True)
        h = (x8[token] @ up[e].cpu().double()) * f64(x_scale)[token, None] * f64(up_scale[e])
        g = h[:, :inner]
        a = torch.nn.functional.silu(g) if kind == "silu" else torch.nn.functional.silu(g) * h[:, inner:]
        off = (3 * (1 + g.abs()) + 12 + 2 * g.abs() + 3 + 3) * EPS32
        a8, a_scale = quantize(a)
        # the row's largest value has the largest part in its scale, whichever of the largest it is
        scale_off = off.amax(1, keepdim=True) + 2 * EPS32
        q = a / f64(a_scale)[:, None]
        near = ((q - q.floor()) - 0.5).abs() <= q.abs() * (off + scale_off + 2 * EPS32) + 1e-30
        d = down[e].cpu().double() * f64(down_scale[e])
        y = (a8 @ d) * f64(a_scale)[:, None]
        y_err = (near.double() @ d.abs()) * f64(a_scale)[:, None] + (scale_off + 6 * EPS32) * y.abs()
        w, w_err = weight[token, j][:, None], weight_err[token, j][:, None]
        out.index_add_(0, token, y * w)
        bound.index_add_(0, token, y_err * (w + w_err) + y.abs() * (w_err + (top_k + 2) * EPS32 * w))
    return out, bound + UNIT[dtype] * (out.abs() + bound) + TINY[dtype]
