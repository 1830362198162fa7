"""Rows of the projection with adapters whose product is held in float32 at a time (host arithmetic, no GPU)."""
import pytest
import torch

from grouped_mm_bf16_amd import _lib, lora


@pytest.mark.parametrize("N", [64, 4096, 1 << 21])
def test_the_product_in_float32_stays_small(N):
    for T in (65, 2048, 2049, 8192, 8193, 100000, 10 ** 7):
        most = lora._rows_at_once(T, N)
        assert most == T or most < T and most % 256 == 0
        assert most <= 2048 or most * N <= 1 << 27


def test_the_gradients_workspace_stays_near_its_operands():
    """Of 1 million rows: 0.54 GB of operands, at most 32 + 32 partial sums of [64, 4096] in float32 for each gradient."""
    size = _lib.load().gmm_lora_grad_workspace_bytes
    rows, K, N, R, L = 1 << 20, 4096, 4096, 64, 8
    operands = 2 * 2 * R * (rows + 8 * (L + 2)) * 2
    partial = 2 * 64 * R * K * 4
    places = 5 * 4 * (rows + 8 * (L + 2)) + (1 << 20)
    peaks = 2 * 32 * L * R * 4
    assert 0 < size(rows, K, N, R, L) <= operands + partial + places + peaks
    for rows in (100, 5000, 131072, 1 << 18, 1 << 20):
        assert size(rows, 512, 512, 16, 4) > 0


def test_rows_too_many_for_gradients_are_refused_before_the_forward_pass(monkeypatch):
    monkeypatch.setattr(lora, "_require_gpu", lambda *tensors: None)


    class Launched(Exception):
        pass

    def launch(x):
        raise Launched

    monkeypatch.setattr(lora, "_guard", launch)
    T = 1 << 21
    x = torch.zeros(1, 8, dtype=torch.bfloat16).expand(T, 8)
    weight, a, b = (torch.zeros(*s, dtype=torch.bfloat16) for s in ((8, 8), (1, 8, 256), (1, 256, 8)))
    adapter = torch.zeros(T, dtype=torch.int32)
    for w in (weight, weight.detach().requires_grad_()):      # no gradient of the adapters is wanted
        with pytest.raises(Launched):
            lora.lora_linear(x, w, a, b, adapter)
    for which in ("a", "b"):
        pair = [a.detach().requires_grad_(which == "a"), b.detach().requires_grad_(which == "b")]
        with pytest.raises(RuntimeError, match="too many rows for gradients"):
            lora.lora_linear(x, weight, *pair, adapter)
        with torch.no_grad(), pytest.raises(Launched):
            lora.lora_linear(x, weight, *pair, adapter)
