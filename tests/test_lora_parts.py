"""Rows of the projection with adapters whose product is held in float32 at a time (host arithmetic, no GPU)."""
import pytest

from grouped_mm_bf16_amd import lora


@pytest.mark.parametrize("N", [64, 4096, 1 << 21])
def test_the_product_in_float32_stays_small(N):
    for T in (65, 2048, 2049, 8192, 8193, 100000):
        most = lora._rows_at_once(T, N)
        assert T <= most or most % 256 == 0 and 2 * ((T - 1) % most + 1) >= most
        assert most <= 2304 or most * N <= 1 << 25
