"""The quotients of the 8-bit rounding on a real MI355X where they are hardest: x / scale within a few 2^-24 of the border between two fp32 numbers of which one is a
whole number and a half.  IEEE's quotient decides which way such a value goes; the kernels' is a reciprocal's product with one correction."""
import pytest
import torch

from grouped_mm_bf16_amd import int8
from oracle import int8_oracle as oracle

pytestmark = pytest.mark.gpu
DEV = "cuda"


def pairs():
    """(x, scale) in float64, every pair of 24-bit numbers whose quotient is that near a border next to n + 1/2, n <= 126: with h = 2 n + 1 the border is M 2^-(k + 2),
    M = h 2^(k + 1) +- 1, and M S = X 2^j + e has one S below 2^j for each small e."""
    found = []
    for h in range(1, 254, 2):
        k = 24 - h.bit_length()
        for M in (h * 2 ** (k + 1) - 1, h * 2 ** (k + 1) + 1):
            for j in (23, 24, 25, 26):
                inverse = pow(M, -1, 2 ** j)
                for e in range(-12, 13):
                    for S in range(e * inverse % 2 ** j, 2 ** 24, 2 ** j):
                        X = (M * S - e) >> j
                        if 2 ** 23 <= S and 2 ** 23 <= X < 2 ** 24:
                            found.append((X * 2.0 ** (j - k - 25), S * 2.0 ** -23))
    return torch.tensor(found, dtype=torch.float64)


def test_next_to_a_half():
    x, scale = pairs().unbind(1)
    assert x.numel() > 2000 and torch.equal(x.float().double(), x) and torch.equal(scale.float().double(), scale)
    # a row's largest value that has the scale: one of those around 127 times it
    largest = (127 * scale).float()
    for _ in range(2):
        low = largest / torch.full_like(largest, 127) < scale.float()
        largest = torch.where(low, torch.nextafter(largest, torch.full_like(largest, float("inf"))), largest)
        high = largest / torch.full_like(largest, 127) > scale.float()
        largest = torch.where(high, torch.nextafter(largest, torch.zeros_like(largest)), largest)
    has = largest / torch.full_like(largest, 127) == scale.float()
    assert has.float().mean() > 0.5
    x, largest = x.float()[has], largest[has]
    for turn in (1.0, 2.0 ** -90, 2.0 ** 100):
        rows = torch.stack([largest, x, -x], 1) * turn
        q, s = oracle.quantize(rows)
        quotient = (rows[:, 1] / s).double()
        assert ((quotient % 1 - 0.5).abs() < 2.0 ** -16).all()      # they are where they should be
        got = int8.quantize_rows(rows.to(DEV))
        assert torch.equal(got.scale.cpu(), s) and torch.equal(got.values.cpu().double(), q)
