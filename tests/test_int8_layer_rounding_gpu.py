"""The 8-bit expert layer on a real MI355X, element by element: its experts' rows and their weighted sums stay in fp32, whatever the number of tokens, and one
rounding to x's type follows.  Every element is held against 64 bits with its own bound: none may be missing, or another's."""
import pytest
import torch

from grouped_mm_bf16_amd import int8, moe
from oracle import int8_oracle as oracle
from oracle import operators_oracle as plain

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF, SF = torch.bfloat16, torch.float16, torch.float32


def layer(T, E, H, inner, kind, dtype=BF, seed=0):
    gen = torch.Generator().manual_seed(seed + 31 * T + H)
    x, z = torch.randn(T, H, generator=gen).to(dtype).to(DEV), torch.randn(T, E, generator=gen).to(DEV)
    up = int8.quantize_columns((torch.randn(E, inner * (2 if kind == "swiglu" else 1), H, generator=gen) * H ** -0.5).to(dtype).to(DEV).transpose(1, 2))
    down = int8.quantize_columns((torch.randn(E, H, inner, generator=gen) * inner ** -0.5).to(dtype).to(DEV).transpose(1, 2))
    return x, z, up, down


def check(x, z, up, down, k, kind, renormalize=True):
    out = int8.moe_forward_int8(x, z, up, down, k, kind, renormalize)
    assert out.dtype == x.dtype and out.shape == x.shape
    want, bound = oracle.layer_within(x, z, up.values, up.scale, down.values, down.scale, k, kind, renormalize)
    plain.assert_within(out, want, bound, f"{tuple(x.shape)} {kind}")
    return out


SHAPES = [(1, 4, 2, 64, 64), (1, 128, 8, 2048, 768), (2, 40, 8, 130, 64), (7, 128, 8, 256, 128), (16, 4, 1, 72, 128), (17, 6, 1, 136, 64), (33, 6, 2, 130, 70),
          (64, 8, 2, 512, 768), (65, 8, 2, 256, 128), (128, 8, 2, 1040, 72), (200, 12, 3, 136, 72), (256, 64, 8, 136, 64), (257, 64, 8, 136, 64), (300, 4, 2, 1031, 320),
          (401, 7, 3, 333, 191), (700, 16, 4, 256, 128), (1500, 4, 2, 512, 1024)]


@pytest.mark.parametrize("kind", ["silu", "swiglu"])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("T,E,k,H,inner", SHAPES)
def test_every_element(T, E, k, H, inner, dtype, kind):
    check(*layer(T, E, H, inner, kind, dtype), k, kind)


@pytest.mark.parametrize("T", [5, 300])
def test_weights_over_all_experts(T):
    x, z, up, down = layer(T, 10, 136, 64, "swiglu")
    check(x, z, up, down, 3, "swiglu", False)


@pytest.mark.parametrize("T", [3, 64, 257, 600])
@pytest.mark.parametrize("H", [128, 131])
def test_experts_rows_beyond_half_precision(T, H):
    """Two experts of opposite rows around 10^5, past fp16's 65504: their sum is in range and finite."""
    x, z, up, down = layer(T, 4, H, 64, "swiglu", HF)
    down = int8.Columns(down.values, down.scale * (2e5 / (down.scale.abs().max() * 127)))
    down.values[1::2] = -down.values[0::2].clamp(min=-127)
    down.scale[1::2] = down.scale[0::2].clone()
    up.values[1::2], up.scale[1::2] = up.values[0::2].clone(), up.scale[0::2].clone()
    z[:] = 0.0
    z[:, 2:] = -50.0
    z[:, 1] = -2.0 ** -9      # nearly equal weights: what is left is 2^-11 of a row
    out = check(x, z, up, down, 2, "swiglu")
    y = oracle.layer(x, z[:, :1], up.values[:1], up.scale[:1], down.values[:1], down.scale[:1], 1, "swiglu")
    assert y.abs().max() > 65504 and torch.isfinite(out).all()


def test_a_token_alone_and_among_many():
    """The same token in batches on either side of every limit: within one rounding of each other."""
    x, z, up, down = layer(700, 16, 256, 128, "swiglu")
    want, bound = oracle.layer_within(x, z, up.values, up.scale, down.values, down.scale, 4, "swiglu")
    for T in (1, 4, 16, 64, 65, 256, 257, 700):
        plain.assert_within(int8.moe_forward_int8(x[:T], z[:T], up, down, 4), want[:T], bound[:T], f"{T} tokens")


@pytest.mark.parametrize("dtype", [BF, HF, SF])
@pytest.mark.parametrize("tokens,k,width,extra", [(1, 1, 1, 0), (3, 2, 7, 0), (5, 8, 8, 0), (70, 9, 100, 3), (33, 32, 1031, 0), (200, 3, 2048, 8), (9, 4, 4100, 1)])
def test_sums_of_rows_in_fp32(tokens, k, width, extra, dtype):
    """The step itself, rows that lie apart among them; a slot whose row does not exist takes no part."""
    gen = torch.Generator().manual_seed(tokens + width)
    slots = tokens * k
    y = torch.randn(slots, width + extra, generator=gen).to(DEV)[:, :width]
    rows = torch.randperm(slots, generator=gen).to(torch.int32)
    weight = torch.rand(slots, generator=gen)
    if slots > 4:
        rows[2], rows[4] = -1, slots
    routing = moe.Routing(None, None, weight.to(DEV), None, rows.to(DEV))
    out = int8._summed(y, routing, tokens, k, dtype)
    there = ((rows >= 0) & (rows < slots)).double()[:, None]
    terms = plain.f64(y)[rows.clamp(0, slots - 1).long()] * weight.double()[:, None] * there
    want, size = terms.reshape(tokens, k, -1).sum(1), terms.abs().reshape(tokens, k, -1).sum(1)
    plain.assert_within(out, want, plain.UNIT[dtype] * want.abs() + plain.TINY[dtype] + (k + 1) * plain.EPS32 * size)
