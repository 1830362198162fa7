"""Gathered 8-bit rows of an operand that has none, on a real MI355X, and of one whose only row lies in a wide matrix."""
import pytest
import torch

from grouped_mm_bf16_amd import int8
from oracle import int8_oracle as oracle
from oracle import operators_oracle as plain

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("K", [100, 101, 112])
@pytest.mark.parametrize("M", [5, 90, 700])
@pytest.mark.parametrize("source", [0, 1])
def test_gathered_from(source, M, K, dtype):
    gen = torch.Generator().manual_seed(M + K)
    a = int8.Rows(torch.randint(-128, 128, (4, 128), generator=gen, dtype=torch.int8).to(DEV)[:source, :K], torch.ones(source, device=DEV))
    b = int8.Columns(torch.randint(-128, 128, (3, 40, K), generator=gen, dtype=torch.int8).to(DEV).transpose(1, 2), torch.ones(3, 40, device=DEV))
    offs = torch.tensor([M // 3, M // 2, M], dtype=torch.int32, device=DEV)
    index = torch.randint(-1, 3, (M,), generator=gen).to(torch.int32).to(DEV)
    out = int8.grouped_int8_mm(a, b, offs, dtype, index)
    if source:
        want, bound, _ = oracle.grouped_mm(a.values, a.scale, b.values, b.scale, offs, dtype, index)
        plain.assert_within(out, want, bound)
    else:
        assert out.shape == (M, 40) and not out.any()
