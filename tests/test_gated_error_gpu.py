"""The activation and its gradient in fp32 on a real MI355X: as near to 64 bits as the formula itself in elementary fp32 operations, or nearer."""
import pytest
import torch

from grouped_mm_bf16_amd import moe_train

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("kind", ["silu", "swiglu"])
@pytest.mark.parametrize("scale", [0.3, 1.0, 4.0])
def test_no_further_off_than_the_formula(kind, scale):
    """What the formula rounds: 1 + e, its reciprocal, two products for the result, five operations more for the gradient of the gate.  A quotient in place of the
    reciprocal and a product is one rounding less; none of the kernel's is one more."""
    rows, inner = 700, 1031
    gen = torch.Generator(device=DEV).manual_seed(1)
    h = torch.randn(rows, inner * (2 if kind == "swiglu" else 1), device=DEV, generator=gen) * scale
    d = torch.randn(rows, inner, device=DEV, generator=gen)

    def formula(h, d):
        gate, up = h[:, :inner], h[:, inner:] if kind == "swiglu" else 1.0
        part = 1 / (1 + (-gate).exp())
        results = [gate * part * up, d * up * (part * (1 + gate * (1 - part)))]
        return results + ([d * gate * part] if kind == "swiglu" else [])

    leaf = h.clone().requires_grad_()
    out = moe_train.gated(leaf, kind)
    grad, = torch.autograd.grad(out, leaf, d)
    own = [out.detach(), grad[:, :inner], grad[:, inner:]]
    for name, got, plain, want in zip(("result", "gate's gradient", "partner's gradient"), own, formula(h, d), formula(h.double(), d.double())):
        off, plain_off = ((t.double() - want).norm() / want.norm() for t in (got, plain))
        assert off <= plain_off, f"{name}: {off:.3g}, the formula {plain_off:.3g}"


def test_far_from_zero():
    """Where e^-g overflows, underflows or is nothing beside one; infinities as the formula has them."""
    g = torch.tensor([-1e30, -200.0, -104.0, -89.0, -88.0, -30.0, -17.0, 0.0, 17.0, 30.0, 88.0, 104.0, 1e4, 1e30, float("inf"), float("nan")], device=DEV)
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        h = g.to(dtype)[None].clone().requires_grad_()
        out = moe_train.gated(h, "silu")
        grad, = torch.autograd.grad(out, h, torch.ones_like(out))
        x = h.detach().double()
        want, want_grad = x * torch.sigmoid(x), torch.sigmoid(x) * (1 + x * torch.sigmoid(-x))
        # rounded once and a few roundings of fp32 in between, those of the exponent by its size; below 2^-126 e^g is lost with its reciprocal
        unit = torch.finfo(dtype).eps / 2
        size = unit + (20 + 2 * x.abs().clamp(max=110)) * 2.0 ** -24
        low = 2.0 ** -126 * x.abs().clamp(1, 110) + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
        for got, exact in ((out, want), (grad, want_grad)):
            fine = torch.isfinite(exact)
            assert ((got.detach().double() - exact).abs() <= size * exact.abs() + low)[fine].all()
        assert out[0, -1].isnan() and grad[0, -1].isnan() and (out[0, -2] == float("inf"))


def test_a_closed_gate_beside_a_large_partner():
    """What a gate far below zero lets through is zero, though the partner's product with its gradient is past fp32's range."""
    for dtype in (torch.float32, torch.bfloat16):
        h = torch.tensor([[-300.0, -1e5, 1e38, -1e38]], device=DEV, dtype=dtype, requires_grad=True)
        out = moe_train.gated(h)
        grad, = torch.autograd.grad(out, h, torch.full_like(out, 1e30))
        assert not out.any() and not grad.any()
