"""Gradients of adapters on a real MI355X from so many rows that a chunk of them is longer than the places that a workgroup holds at a time."""
import pytest
import torch

from test_lora_gpu import BF, DEV, HF, check_grads, make

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
