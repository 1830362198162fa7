"""64-bit restatements of the operators around the grouped product, on the CPU, from their formulas: layer norm, the projection with
low-rank adapters, the expert layer.  Used by the tests only; independent of the package."""
import torch

UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}   # of one rounding to nearest
TINY = {torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24, torch.float32: 2.0 ** -149}  # smallest step
EPS32 = 2.0 ** -24


def f64(t):
    return None if t is None else t.detach().cpu().double()


def assert_within(got, want, bound, what=""):
    """|got - want| <= bound elementwise, where want is finite; the same infinities and NaN elsewhere."""
    got = f64(got)
    assert got.shape == want.shape, f"{what}: shape {tuple(got.shape)}, not {tuple(want.shape)}"
    fine = torch.isfinite(want)
    same = torch.where(fine, torch.isfinite(got), (got == want) | (got.isnan() & want.isnan()))
    assert same.all(), f"{what}: {int((~same).sum())} values are finite where they should not be, or the other way round"
    off = torch.where(fine, (got - want).abs() - bound, torch.zeros_like(want))
    at = off.argmax() if off.numel() else None
    assert at is None or off.flatten()[at] <= 0, (
        f"{what}: element {int(at)} is {got.flatten()[at]:.9g}, not {want.flatten()[at]:.9g}; allowed {(bound + torch.zeros_like(want)).flatten()[at]:.3g}")


# ------------------------------------------------------------------ layer norm
def layer_norm(x, weight=None, bias=None, eps=1e-5):
    x = f64(x)
    z = x - x.mean(-1, keepdim=True)
    z = z / (z.square().mean(-1, keepdim=True) + eps).sqrt()
    y = z if weight is None else z * f64(weight)
    return y if bias is None else y + f64(bias)


def layer_norm_backward(dy, x, weight=None, eps=1e-5):
    """dx, dweight, dbias for rows x [rows, width]."""
    dy, x = f64(dy), f64(x)
    mean = x.mean(-1, keepdim=True)
    rstd = 1 / ((x - mean).square().mean(-1, keepdim=True) + eps).sqrt()
    z = (x - mean) * rstd
    g = dy if weight is None else dy * f64(weight)
    dx = rstd * (g - g.mean(-1, keepdim=True) - z * (g * z).mean(-1, keepdim=True))
    return dx, (dy * z).sum(0), dy.sum(0)


def layer_norm_bounds(dy, x, weight, bias, eps, dtype, param_dtype):
    """Bounds of y, dx, dweight, dbias (y's alone without dy): one rounding of the result to its type (of the terms' size where they
    cancel), and fp32 arithmetic in between, whose sums are of at
    most 64 terms one after the other and then of a tree, or of `rows` terms."""
    x = f64(x)
    mean = x.mean(-1, keepdim=True)
    rstd = 1 / ((x - mean).square().mean(-1, keepdim=True) + eps).sqrt()
    z = ((x - mean) * rstd).abs()
    w = torch.ones(x.size(-1), dtype=torch.float64) if weight is None else f64(weight).abs()
    b = torch.zeros(x.size(-1), dtype=torch.float64) if bias is None else f64(bias).abs()
    sum_err = 80 * EPS32
    z_err = sum_err * (x.abs().mean(-1, keepdim=True) * rstd + z * (1 + x.abs().mean(-1, keepdim=True) * rstd)) + 4 * EPS32 * x.abs() * rstd
    y = layer_norm(x, weight, bias, eps).abs()
    bounds = [UNIT[dtype] * y + TINY[dtype] + z_err * w + 4 * EPS32 * (z * w + b)]
    if dy is None:
        return bounds[0]
    dy = f64(dy).abs()
    g = dy * w
    c1, c2 = g.mean(-1, keepdim=True), (g * z).mean(-1, keepdim=True)
    c2_err = sum_err * c2 + (g * z_err).mean(-1, keepdim=True)
    dx_err = rstd * (8 * EPS32 * (g + c1 + z * c2) + sum_err * c1 + z * c2_err + z_err * c2 + sum_err * (g + c1 + z * c2))
    rows = x.size(0)
    col_err = (rows + 64) * EPS32
    return [bounds[0], UNIT[dtype] * (rstd * (g + c1 + z * c2)) + TINY[dtype] + dx_err,
            UNIT[param_dtype] * (dy * z).sum(0) + TINY[param_dtype] + col_err * (dy * z).sum(0) + (dy * z_err).sum(0),
            UNIT[param_dtype] * dy.sum(0) + TINY[param_dtype] + col_err * dy.sum(0)]


# ------------------------------------------------------------------ expert layer
def moe_layer(x, logits, w_up, w_down, top_k, kind, renormalize=True):
    """out, and its bound for a kernel that holds everything in between in 32 bits or as two 16-bit values and rounds once.
    kind: "silu", "swiglu", "interleaved"."""
    x, z, dtype = f64(x), f64(logits), x.dtype
    order = torch.argsort(z, dim=1, descending=True, stable=True)[:, :top_k]
    top = z.gather(1, order)
    best = z.max(1, keepdim=True).values
    if renormalize:
        weight = torch.softmax(top, 1)
    else:
        weight = torch.exp(top - best) / torch.exp(z - best).sum(1, keepdim=True)
    odd = torch.isinf(best)[:, 0]        # all weight, in equal shares, on what equals the maximum
    if odd.any():
        at = (top == best).double()
        among = at.sum(1, keepdim=True) if renormalize else (z == best).double().sum(1, keepdim=True)
        weight[odd] = (at / among)[odd]
    two16 = {torch.bfloat16: 2.0 ** -15, torch.float16: 2.0 ** -21}[dtype]
    H, I = x.size(1), w_down.size(1)
    out, bound = torch.zeros_like(x), torch.zeros_like(x)
    for e in order.unique().tolist():
        token, choice = (order == e).nonzero(as_tuple=True)
        U, D = f64(w_up[e]), f64(w_down[e])
        h, h_abs = x[token] @ U, x[token].abs() @ U.abs()
        h_err = (H / 16 + 40) * EPS32 * h_abs
        if kind == "silu":
            act = h * torch.sigmoid(h)
            err = 1.1 * h_err + 32 * EPS32 * act.abs()
        else:
            c = torch.arange(I)
            gate = c if kind == "swiglu" else c // 64 * 128 + c % 64
            up = gate + (I if kind == "swiglu" else 64)
            s = h[:, gate] * torch.sigmoid(h[:, gate])
            act = s * h[:, up]
            err = 1.1 * h_err[:, gate] * h[:, up].abs() + s.abs() * h_err[:, up] + 1.1 * h_err[:, gate] * h_err[:, up] + 32 * EPS32 * act.abs()
        err = err + two16 * act.abs() + TINY[dtype]
        w = weight[token, choice][:, None]
        y_err = err @ D.abs() + (I / 16 + 60 + 2.0 ** 6) * EPS32 * (act.abs() @ D.abs())
        out.index_add_(0, token, (act @ D) * w)
        bound.index_add_(0, token, y_err * w + (act @ D).abs() * w * 2.0 ** -17)
    return out, bound + UNIT[dtype] * out.abs() + TINY[dtype]


# ------------------------------------------------------------------ projection with low-rank adapters
def lora_linear(x, weight, lora_a, lora_b, adapter, scale=None, dtype=None):
    """out and its bound: one rounding of the result, for more than 64 rows one of weight's product before it; fp32 sums; the rank-sized
    product as two 16-bit values."""
    dtype, many = dtype or x.dtype, x.size(0) > 64
    x, weight, a, b = f64(x), f64(weight), f64(lora_a), f64(lora_b)
    two16 = {torch.bfloat16: 2.0 ** -15, torch.float16: 2.0 ** -21}[dtype]
    K, R = x.size(1), a.size(2)
    base = x @ weight
    err = (K / 16 + 80) * EPS32 * (x.abs() @ weight.abs()) + (UNIT[dtype] * base.abs() if many else 0)
    out = base.clone()
    for i in adapter.cpu().unique().tolist():
        if not 0 <= i < a.size(0):
            continue
        at = (adapter.cpu() == i).nonzero()[:, 0]
        s = 1.0 if scale is None else float(scale[i])
        low = x[at] @ a[i]
        low_err = (K / 16 + 80) * EPS32 * (x[at].abs() @ a[i].abs()) + (two16 + 4 * EPS32) * low.abs() + TINY[dtype] / max(abs(s), 1e-30)
        out[at] += s * (low @ b[i])
        err[at] += abs(s) * (low_err @ b[i].abs() + (R + 8) * EPS32 * (low.abs() @ b[i].abs()))
    return out, err * (1 + UNIT[dtype]) + UNIT[dtype] * out.abs() + TINY[dtype]


def lora_backward(dy, x, weight, lora_a, lora_b, adapter, scale=None, dtype=None):
    """(dx, its bound), (dweight, ..), (da, ..), (db, ..)."""
    dtype = dtype or x.dtype
    dx = lora_linear(dy, weight.mT, lora_b.mT, lora_a.mT, adapter, scale, dtype)
    dy, x, a, b = f64(dy), f64(x), f64(lora_a), f64(lora_b)
    two16 = {torch.bfloat16: 2.0 ** -15, torch.float16: 2.0 ** -21}[dtype]
    T, K, N = x.size(0), x.size(1), dy.size(1)
    dw = x.T @ dy
    dw_err = (T + 80) * EPS32 * (x.abs().T @ dy.abs())
    da, db, da_err, db_err = (torch.zeros_like(t) for t in (a, b, a, b))
    for i in adapter.cpu().unique().tolist():
        if not 0 <= i < a.size(0):
            continue
        at = (adapter.cpu() == i).nonzero()[:, 0]
        s = 1.0 if scale is None else float(scale[i])
        low, u = x[at] @ a[i], dy[at] @ b[i].T
        low_err = abs(s) * (K / 16 + 80) * EPS32 * (x[at].abs() @ a[i].abs()) + (two16 + 4 * EPS32) * abs(s) * low.abs() + TINY[dtype]
        u_err = abs(s) * (N / 16 + 80) * EPS32 * (dy[at].abs() @ b[i].abs().T) + (two16 + 4 * EPS32) * abs(s) * u.abs() + TINY[dtype]
        rows = (len(at) / 16 + 80) * EPS32
        da[i], db[i] = s * (x[at].T @ u), s * (low.T @ dy[at])
        da_err[i] = x[at].abs().T @ u_err + rows * abs(s) * (x[at].abs().T @ u.abs())
        db_err[i] = low_err.T @ dy[at].abs() + rows * abs(s) * (low.abs().T @ dy[at].abs())
    return dx, *((v, e + UNIT[dtype] * v.abs() + TINY[dtype]) for v, e in ((dw, dw_err), (da, da_err), (db, db_err)))
