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
