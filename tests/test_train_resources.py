"""What the compiler made of the kernels of trained and 8-bit expert layers and of dropout (metadata of the built library, no GPU needed):
everything in registers."""
import re

from test_kernel_resources import kernels  # noqa: F401  (the fixture)


def test_no_scratch_memory(kernels):  # noqa: F811
    own = {n: k for n, k in kernels.items() if re.search(r"sort_rows|sum_rows|combine_backward|route_backward|gated_kernel|dropout_kernel|quantize_kernel|GmmInt8Params", n)}
    assert len(own) > 50
    assert {n: k[".private_segment_fixed_size"] for n, k in own.items() if k[".private_segment_fixed_size"]} == {}
