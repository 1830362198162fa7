"""The projection with adapters on a real MI355X where the rank-sized values are far from one: they are held to the range and precision of
float32, in half precision too, whatever the number of rows."""
import pytest
import torch

from grouped_mm_bf16_amd import lora
from oracle import operators_oracle as oracle
from test_lora_gpu import BF, DEV, HF, make, matrix

pytestmark = pytest.mark.gpu
EPS = oracle.EPS32
TWO16 = {BF: 2.0 ** -15, HF: 2.0 ** -21}      # of a value held as two 16-bit ones
FLOOR = 2.0 ** -38                            # of the largest of the values that share a power of two


def bound_of(x, weight, a, b, adapter, scale):
    """out and its bound as the oracle has it, with one rounding of the result, and for x @ a no other error than a relative one."""
    want, _ = oracle.lora_linear(x, weight, a, b, adapter, scale)
    dtype = x.dtype
    x, weight, a, b = oracle.f64(x), oracle.f64(weight), oracle.f64(a), oracle.f64(b)
    K, R = x.size(1), a.size(2)
    err = (K / 16 + 80) * EPS * (x.abs() @ weight.abs())
    for i in adapter.cpu().unique().tolist():
        if not 0 <= i < a.size(0):
            continue
        at, s = (adapter.cpu() == i).nonzero()[:, 0], float(scale[i])
        low = (x[at] @ a[i]).abs()
        low_err = (K / 16 + 80) * EPS * (x[at].abs() @ a[i].abs()) + (TWO16[dtype] + 4 * EPS) * low + FLOOR * low.max(1, keepdim=True).values
        err[at] += s * (low_err @ b[i].abs() + (R + 8) * EPS * (low @ b[i].abs()))
    unit = oracle.UNIT[dtype]
    return want, err * (1 + unit) + unit * want.abs() + oracle.TINY[dtype]


def check_range(x, weight, a, b, adapter, scale):
    want, bound = bound_of(x, weight, a, b, adapter, scale)
    assert torch.isfinite(want).all() and want.abs().max() < 60000
    oracle.assert_within(lora.lora_linear(x, weight, a, b, adapter, scale), want, bound, "out")
    return want


@pytest.mark.parametrize("T", [6, 100, 256, 257, 400])
@pytest.mark.parametrize("R,lay", [(16, "rows"), (16, "cols"), (72, "rows"), (136, "cols"), (5, "any")])
def test_rank_sized_values_past_65504(T, R, lay):
    x, weight, a, b, adapter, scale = make(T, 128, 96, R, 3, lay, "rows", HF)
    x, a, b = x.abs() * 8 + 8, a.abs() * 100 + 50, b * 2.0 ** -10
    want = check_range(x, weight, a, b, adapter, scale)
    assert ((oracle.f64(x) @ oracle.f64(a[0])) > 65504).any() and want.abs().max() > 1


@pytest.mark.parametrize("T", [6, 100, 257, 400])
@pytest.mark.parametrize("size", [-12, -18, -22])
@pytest.mark.parametrize("R,lay", [(16, "rows"), (16, "cols"), (72, "rows"), (136, "cols")])
def test_small_rank_sized_values(T, size, R, lay):
    """x and A small, B large: x @ A is some 2^size, the result is not."""
    gen = torch.Generator().manual_seed(T + size)
    _, _, _, _, adapter, scale = make(T, 8, 8, 8, 3)
    x = (torch.randn(T, 128, generator=gen) * 2.0 ** (size // 2)).to(HF).to(DEV)
    a = matrix(gen, (3, 128, R), HF, 2.0 ** (size - size // 2 - 3), lay)
    b = matrix(gen, (3, R, 96), HF, 1000.0, lay)
    want = check_range(x, torch.zeros(128, 96, dtype=HF, device=DEV), a, b, adapter, scale)
    assert want.abs().max() > 2.0 ** -14


def test_rows_of_very_different_size_beside_one_another():
    """A strip of rows whose x @ A span sixteen powers of ten, zeros among them, in both types."""
    for dtype, size in ((HF, 4), (BF, 8)):
        x, weight, a, b, adapter, scale = make(400, 128, 96, 16, 2, dtype=dtype)
        weight = torch.zeros_like(weight)
        x = (x.float() * 10.0 ** (torch.arange(400) % (2 * size + 1) - size).to(DEV)[:, None]).to(dtype)
        x[7::16] = 0
        a = a * 0.5
        want, bound = bound_of(x, weight, a, b, adapter, scale)
        oracle.assert_within(lora.lora_linear(x, weight, a, b, adapter, scale), want, bound, str(dtype))


@pytest.mark.parametrize("T", [100, 400])
def test_infinities_stay_in_their_rows_of_half_precision(T):
    x, weight, a, b, adapter, scale = make(T, 128, 64, 8, 2, dtype=HF)
    adapter[:] = 0
    want = lora.lora_linear(x, weight, a, b, adapter, scale)
    x[3, 5] = float("inf")
    got = lora.lora_linear(x, weight, a, b, adapter, scale)
    keep = torch.arange(T, device=DEV) != 3
    assert torch.equal(got[keep], want[keep]) and not torch.isfinite(got[3]).any()
