"""What the compiler made of the kernels of layer norm, of projections with adapters and of the few-token expert layer (metadata of the
built library, no GPU needed): everything in registers, but for the backward pass of the longest rows."""
import re

from test_kernel_resources import kernels  # noqa: F401  (the fixture)


def test_operators_use_no_scratch_memory(kernels):  # noqa: F811
    own = {n: k for n, k in kernels.items() if re.search(r"lora_|few_|norm_", n)}
    assert len(own) > 150
    scratch = {n: k[".private_segment_fixed_size"] for n, k in own.items() if k[".private_segment_fixed_size"]}
    # rows of 8193 to 16384 elements, 32 to a lane, with the sums of both parameters' gradients: a few registers of 16-bit rows, more of fp32
    longest = {n for n in scratch if "norm_backward_kernel" in n and re.search(r"Li8ELi512ELi4E|Li4ELi512ELi8E", n)}
    assert set(scratch) == longest
    assert all(scratch[n] <= (192 if "IfLi4" in n else 24) for n in longest)
