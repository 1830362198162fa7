"""The 8-bit expert layer past the 2 GiB of 8-bit rows that one gathered product takes, on a real MI355X: any number of tokens."""
import pytest
import torch

from grouped_mm_bf16_amd import int8
from oracle import int8_oracle as oracle
from oracle import operators_oracle as plain

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = torch.bfloat16


@pytest.mark.parametrize("T,H,inner,kind", [(16390, 131056, 16, "swiglu"), (33000, 131000, 64, "swiglu"), (20001, 107375, 33, "silu")])
def test_tokens_past_two_gibibytes(T, H, inner, kind):
    assert T * H > 2 ** 31 - 2 ** 18
    gen = torch.Generator(device=DEV).manual_seed(T)
    x = torch.randn(T, H, device=DEV, dtype=BF, generator=gen)
    z = torch.randn(T, 2, device=DEV, generator=gen)
    weight = lambda *shape: torch.randn(*shape, device=DEV, dtype=BF, generator=gen).mul_(shape[-2] ** -0.5)
    up, down = int8.quantize_columns(weight(2, H, inner * (2 if kind == "swiglu" else 1))), int8.quantize_columns(weight(2, inner, H))
    out = int8.moe_forward_int8(x, z, up, down, 1, kind)
    assert out.shape == x.shape
    rows = torch.tensor([0, 1, T // 3, T // 2 - 1, T // 2, T // 2 + 1, 2 * T // 3, T - 2, T - 1])
    want, bound = oracle.layer_within(x[rows.to(DEV)], z[rows.to(DEV)], up.values, up.scale, down.values, down.scale, 1, kind)
    plain.assert_within(out[rows.to(DEV)], want, bound)
    if kind == "swiglu" and inner % 64:      # (the epilogue's activation has other last bits than that of a smaller batch)
        for first in (0, T // 2 - 200, T - 400):
            part = slice(first, first + 400)
            assert torch.equal(out[part], int8.moe_forward_int8(x[part], z[part], up, down, 1, kind))
