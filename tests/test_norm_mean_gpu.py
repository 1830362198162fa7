"""Layer norm on a real MI355X of rows whose mean is far from zero: the mean's own rounding must not show in the result, whatever the width."""
import pytest
import torch

from grouped_mm_bf16_amd import norm
from oracle import operators_oracle as oracle
from test_norm_gpu import BF, DEV, HF, SF, make

pytestmark = pytest.mark.gpu
EPS = oracle.EPS32

WIDTHS = [3, 7, 65, 100, 329, 513, 1000, 1031, 1536, 3001, 5120, 7168, 8199, 14337]


@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("dtype", [BF, HF, SF])
def test_constant_rows(width, dtype):
    """x - mean is zero.  The mean that a sum in fp32 gives is 80 roundings off at most; taken again of what is left, 80 roundings of that."""
    values = torch.tensor([3.0, -1e4, 0.1, 60000.0, -777.0, 1.0, 4097.0]).to(dtype)
    x = values[:, None].expand(-1, width).contiguous().to(DEV)
    _, dy, w, b = make(len(values), width, dtype, dtype, width)
    off = (80 * EPS) ** 2 * oracle.f64(values).abs()[:, None] * 1e-5 ** -0.5
    got = norm.layer_norm(x, w, b)
    want = oracle.f64(b).expand(len(values), width)
    oracle.assert_within(got, want, oracle.UNIT[dtype] * want.abs() + (1 + 2.0 ** -7) * off * oracle.f64(w).abs() + 4 * EPS, "y")
    # z is zero in the backward pass too
    leaves = [t.detach().requires_grad_() for t in (x, w, b)]
    dx, dw, _ = torch.autograd.grad(norm.layer_norm(*leaves), leaves, dy)
    oracle.assert_within(dw, torch.zeros(width, dtype=torch.float64), (off * oracle.f64(dy).abs()).sum(0) * 1.01 + oracle.TINY[dtype], "dweight")
    assert torch.isfinite(dx).all()


@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("mean", [4096.0, -1e4, 1e5])
def test_large_means_in_float32(width, mean):
    """x - mean is exact to a rounding or two of x - mean and of the correction."""
    gen = torch.Generator().manual_seed(width)
    x = (mean + torch.randn(5, width, generator=gen)).to(DEV)
    d = oracle.f64(x) - oracle.f64(x).mean(1, keepdim=True)
    rstd = 1 / (d.square().mean(1, keepdim=True) + 1e-5).sqrt()
    # the first mean: 80 roundings of its size, all of which the second sum takes back but 80 roundings of what it adds up
    first = 80 * EPS * abs(mean)
    off = (8 * EPS * (d.abs() + first) + 80 * EPS * (d.abs().mean(1, keepdim=True) + first)) * rstd
    bound = off * (1 + (d * rstd).abs()) + 200 * EPS * (d * rstd).abs()
    oracle.assert_within(norm.layer_norm(x), d * rstd, bound, "y")
