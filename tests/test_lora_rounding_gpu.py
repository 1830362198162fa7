"""The projection with many requests' adapters on a real MI355X: its results, and the gradients of its input, are rounded once whatever the
number of rows."""
import pytest
import torch

from grouped_mm_bf16_amd import _lib, lora
from oracle import operators_oracle as oracle
from test_lora_gpu import BF, DEV, HF, check, check_grads, make

pytestmark = pytest.mark.gpu


def of_one_rounding(bound, x, weight):
    """The oracle's bound without what it allows more than 64 rows for a rounding of x @ weight before the adapters' part."""
    return bound - oracle.UNIT[x.dtype] * (1 + oracle.UNIT[x.dtype]) * (oracle.f64(x) @ oracle.f64(weight)).abs()


@pytest.mark.parametrize("T", [65, 256, 257, 400, 1025])
@pytest.mark.parametrize("K,N,R,lay", [(256, 192, 16, "rows"), (264, 136, 40, "cols"), (136, 261, 100, "rows"), (96, 77, 5, "cols"),
                                       (64, 5, 8, "rows"), (72, 80, 12, "any")])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_many_rows_are_rounded_once(T, K, N, R, lay, dtype):
    for pattern in ("mixed", "requests", "none"):
        x, weight, a, b, adapter, scale = make(T, K, N, R, 4, lay, "rows", dtype, pattern)
        want, bound = oracle.lora_linear(x, weight, a, b, adapter, scale)
        oracle.assert_within(lora.lora_linear(x, weight, a, b, adapter, scale), want, of_one_rounding(bound, x, weight), pattern)
    want, bound = oracle.lora_linear(x, weight, a[:0], b[:0], adapter, scale[:0])
    oracle.assert_within(lora.lora_linear(x, weight, a[:0], b[:0], adapter, scale[:0]), want, of_one_rounding(bound, x, weight), "no adapters")


@pytest.mark.parametrize("T", [100, 300])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_the_gradient_of_many_rows_is_rounded_once(T, dtype):
    x, weight, a, b, adapter, scale = make(T, 200, 136, 16, 3, dtype=dtype)
    dy = torch.randn(T, 136, generator=torch.Generator().manual_seed(T)).to(dtype).to(DEV)
    leaf = x.detach().requires_grad_()
    got, = torch.autograd.grad(lora.lora_linear(leaf, weight, a, b, adapter, scale), leaf, dy)
    want, bound = oracle.lora_backward(dy, x, weight, a, b, adapter, scale)[0]
    oracle.assert_within(got, want, of_one_rounding(bound, dy, weight.t()), "dx")


@pytest.mark.parametrize("most", [256, 300, 640])
def test_rows_taken_in_parts(most, monkeypatch):
    """The product in float32 is held for a part of the rows at a time; forward, and what the backward pass takes from it."""
    monkeypatch.setattr(lora, "_rows_at_once", lambda rows, columns: most)
    x, weight, a, b, adapter, scale = make(1001, 264, 200, 16, 5, pad=3)
    check(x, weight, a, b, adapter, scale)
    check_grads(x, weight, a, b, adapter, scale)


def test_adapters_added_to_a_rounded_product():
    """gmm_lora_add: the product lies in the result's place already, rounded."""
    for T, N, lay in ((40, 192, "rows"), (200, 96, "cols"), (400, 192, "rows"), (300, 203, "cols"), (300, 5, "rows")):
        x, weight, a, b, adapter, scale = make(T, 256, N, 16, 4, lay)
        out = (x.float() @ weight.float()).to(BF)
        want, bound = oracle.lora_linear(x, weight, a, b, adapter, scale)
        extra = oracle.UNIT[BF] * (1 + oracle.UNIT[BF]) * (oracle.f64(x) @ oracle.f64(weight)).abs() if T <= 64 else 0
        lib = _lib.load()
        nbytes = lib.gmm_lora_workspace_bytes(T, 256, N, 16)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=DEV)
        rc = lib.gmm_lora_add(x.data_ptr(), a.data_ptr(), b.data_ptr(), adapter.data_ptr(), scale.data_ptr(), out.data_ptr(), None, T, 256, N,
                              16, 4, x.stride(0), *a.stride(), *b.stride(), N, _lib.DT_BF16, ws.data_ptr(), nbytes,
                              torch.cuda.current_stream().cuda_stream)
        assert rc == 0
        oracle.assert_within(out, want, bound + extra, f"{T} rows")
