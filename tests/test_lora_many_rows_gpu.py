"""Gradients of adapters on a real MI355X from so many rows that a chunk of them is longer than the places that a workgroup holds at a time."""
import pytest
import torch

from grouped_mm_bf16_amd import lora
from oracle import operators_oracle as oracle
from test_lora_gpu import BF, DEV, HF, check_grads, make
from test_lora_rounding_gpu import of_one_rounding

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [135000, 150001])
@pytest.mark.parametrize("dtype,R", [(BF, 8), (HF, 20)])
def test_gradients(T, dtype, R):
    x, weight, a, b, adapter, scale = make(T, 24, 40, R, 3, dtype=dtype, pattern="requests")
    check_grads(x, weight, a, b, adapter, scale)


def test_one_adapter_has_nearly_all_rows():
    x, weight, a, b, adapter, scale = make(140000, 16, 24, 8, 4)
    adapter = torch.where(torch.rand(140000, generator=torch.Generator().manual_seed(0)).to(DEV) < 1e-3, adapter, 2).to(torch.int32)
    check_grads(x, weight, a, b, adapter, scale)


def test_columns_fewer_than_eight():
    check_grads(*make(136000, 5, 24, 4, 2))


def test_rows_past_what_is_held_at_a_time():
    """[8232, 16384] of float32 are more than 512 MiB: two parts, the second of a few rows."""
    T, N = 8192 + 40, 16384
    x, weight, a, b, adapter, scale = make(T, 64, N, 8, 3, pattern="requests")
    assert lora._rows_at_once(T, N) == 8192
    got = lora.lora_linear(x, weight, a, b, adapter, scale)
    keep = [0, 1, 4000, 8190, 8191, 8192, 8193, 8200, T - 1]
    keep += list(range(100, 8192, 128))[:70 - len(keep)]
    at = torch.tensor(keep, device=DEV)
    want, bound = oracle.lora_linear(x[at], weight, a, b, adapter[at], scale)
    oracle.assert_within(got[at], want, of_one_rounding(bound, x[at], weight))
