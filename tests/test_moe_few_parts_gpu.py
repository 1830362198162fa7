"""The expert layer for a few tokens on a real MI355X where the second product's workgroups keep the most activations that they may: 16 rows
of 1024, more than 64 KB of LDS."""
import pytest

from test_moe_few_gpu import BF, HF, check, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [15, 16])
@pytest.mark.parametrize("I", [8192, 8100])
@pytest.mark.parametrize("lay,kind,dtype", [("rows", "swiglu", BF), ("cols", "swiglu", HF), ("rows", "silu", HF), ("padded", "silu", BF)])
def test_one_expert(T, I, lay, kind, dtype):
    check(*make(T, 1, 1024, I, kind, lay, dtype), 1, kind)


@pytest.mark.parametrize("lay", ["rows", "cols"])
def test_four_experts(lay):
    check(*make(16, 4, 2048, 4096, "interleaved", lay), 1, "interleaved")
