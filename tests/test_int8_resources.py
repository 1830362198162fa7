"""What the compiler made of the 8-bit products' kernels for few rows, of their sums and of the counted routing (metadata of the built library, no GPU needed):
everything in registers."""
from test_kernel_resources import kernels  # noqa: F401  (the fixture)

NAMES = ("int8_few_kernel", "int8_combine_kernel", "int8_finish_kernel", "moe_place_counted_kernel", "sum_rows_kernel")


def test_no_scratch_memory(kernels):  # noqa: F811
    own = {n: k for n, k in kernels.items() if any(name in n for name in NAMES)}
    for name in NAMES:
        assert any(name in n for n in own), name
    assert {n: k[".private_segment_fixed_size"] for n, k in own.items() if k[".private_segment_fixed_size"]} == {}

