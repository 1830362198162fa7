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


# ------------------------------------------------------------------ gradients of the adapters
def grad_bounds(dy, x, a, b, adapter, scale):
    """(da, its bound), (db, its bound): one rounding, sums in float32, and of the values that are held as two 16-bit ones a relative error."""
    dtype = x.dtype
    dy, x, a, b = oracle.f64(dy), oracle.f64(x), oracle.f64(a), oracle.f64(b)
    (T, K), N = x.shape, dy.size(1)
    da, db, da_err, db_err = (torch.zeros_like(t) for t in (a, b, a, b))
    for i in adapter.cpu().unique().tolist():
        if not 0 <= i < a.size(0):
            continue
        at, s = (adapter.cpu() == i).nonzero()[:, 0], float(scale[i])
        sums = (len(at) / 16 + 80) * EPS
        for p, q, m, size, out, err in ((x[at], dy[at] @ b[i].T, dy[at].abs() @ b[i].abs().T, N, da, da_err),
                                        (dy[at], x[at] @ a[i], x[at].abs() @ a[i].abs(), K, db, db_err)):
            q_err = s * ((size / 16 + 80) * EPS * m + (TWO16[dtype] + 4 * EPS) * q.abs() + FLOOR * q.abs().max(0).values)
            value, bound = s * (p.T @ q), p.abs().T @ q_err + sums * s * (p.abs().T @ q.abs())
            out[i], err[i] = (value, bound) if out is da else (value.T, bound.T)
    unit = oracle.UNIT[dtype]
    return [(v, e * (1 + unit) + unit * v.abs() + oracle.TINY[dtype]) for v, e in ((da, da_err), (db, db_err))]


def check_adapter_grads(dy, x, a, b, adapter, scale, least):
    weight = torch.zeros(x.size(1), dy.size(1), dtype=x.dtype, device=DEV)
    leaves = [t.detach().requires_grad_() for t in (a, b)]
    got = torch.autograd.grad(lora.lora_linear(x, weight, *leaves, adapter, scale), leaves, dy)
    for name, g, (want, bound), low in zip(("da", "db"), got, grad_bounds(dy, x, a, b, adapter, scale), least):
        assert torch.isfinite(want).all() and low < want.abs().max() < 60000
        oracle.assert_within(g, want, bound, name)


@pytest.mark.parametrize("T", [40, 300, 1500])
@pytest.mark.parametrize("R,lay", [(16, "rows"), (5, "cols"), (72, "cols"), (256, "rows"), (1, "rows")])
@pytest.mark.parametrize("size", [1e-5, 1e-6])
def test_gradients_of_small_gradients(T, R, lay, size):
    """A first step of tuning: dy as it is without loss scaling, B of 0.02.  dB is of the size of dy, so its adapters get a large A."""
    x, _, a, b, adapter, scale = make(T, 136, 256, R, 3, lay, "rows", HF)
    dy = (torch.randn(T, 256, generator=torch.Generator().manual_seed(5)) * size).to(HF).to(DEV)
    check_adapter_grads(dy, x * 64, a * 64, b * 0.02 * R ** 0.5, adapter, scale, (size, size))


@pytest.mark.parametrize("T", [40, 300, 1500])
def test_gradients_of_rank_sized_values_past_65504(T):
    x, _, a, b, adapter, scale = make(T, 128, 96, 16, 3, dtype=HF)
    dy = torch.randn(T, 96, generator=torch.Generator().manual_seed(5)).to(HF).to(DEV)
    large, small = 30000.0, 2.0 ** -12
    check_adapter_grads(dy * 4, x * small, a, b * large, adapter, scale, (1, 0))       # u = dy B^T
    check_adapter_grads(dy * small, x * 4, a * large, b, adapter, scale, (0, 1))       # low = x A


def test_gradients_of_requests_of_very_different_size():
    """Each adapter's rows have a power of two of their own: one's large gradients do not take another's bits."""
    x, _, a, b, adapter, scale = make(900, 64, 96, 8, 5, dtype=HF, pattern="requests")
    dy = torch.randn(900, 96, generator=torch.Generator().manual_seed(5))
    dy = (dy * 10.0 ** (adapter.cpu().float() * 2 - 6)[:, None]).to(HF).to(DEV)
    check_adapter_grads(dy, x, a, b, adapter, scale, (1, 1))


def test_gradients_of_no_rows_in_half_precision():
    x, weight, a, b, adapter, scale = make(0, 64, 32, 8, 3, dtype=HF)
    leaves = [t.detach().requires_grad_() for t in (a, b)]
    torch.full((1 << 20,), float("nan"), device=DEV)      # what a workspace may be given next
    grads = torch.autograd.grad(lora.lora_linear(x, weight, *leaves, adapter, scale).sum(), leaves)
    assert all(torch.equal(g, torch.zeros_like(g)) for g in grads)
