"""Gathered rows of an operand that has none: every row_index lies outside it, so every row reads as zeros.  What the kernels take for the operand's length is host
arithmetic, held here without a GPU."""
import os
import shutil
import subprocess

import pytest
import torch

from grouped_mm_bf16_amd import int8

HEADER = os.path.abspath(os.path.join(os.path.dirname(__file__), "..", "grouped_mm_bf16_amd", "csrc", "gmm_sched.h"))


def test_bytes_of_rows(tmp_path):
    """Up to the last row's last element, for any pitch; none for no rows (one row's length less a pitch would be a number below zero, and read as nearly
    4 GiB without a sign)."""
    compiler = shutil.which("g++") or shutil.which("c++")
    assert compiler, "a host compiler builds the package too"
    program = tmp_path / "bytes.cpp"
    program.write_text(f'#include <cstdio>\n#include <cstdlib>\n#include "{HEADER}"\n'
                       'int main(int n, char** v) { for (int i = 1; i + 2 < n; i += 3) std::printf("%lld\\n", (long long)gmm_rows_bytes(atoll(v[i]), atoll(v[i + 1]), atoll(v[i + 2]))); }\n')
    subprocess.run([compiler, "-std=c++17", "-o", str(tmp_path / "bytes"), str(program)], check=True)
    cases = [(rows, ld, K) for rows in (0, 1, 2, 70, 100000) for ld, K in ((56, 50), (50, 50), (64, 8), (0, 50), (8192, 8))]
    out = subprocess.run([str(tmp_path / "bytes"), *(str(v) for case in cases for v in case)], check=True, capture_output=True, text=True).stdout.split()
    assert [int(v) for v in out] == [2 * ((rows - 1) * ld + K) if rows else 0 for rows, ld, K in cases]


@pytest.mark.parametrize("K", [100, 112, 101])
@pytest.mark.parametrize("M", [5, 90])
def test_zeros(monkeypatch, M, K):
    monkeypatch.setattr(int8, "_require_gpu", lambda *tensors: None)
    monkeypatch.setattr(int8, "_guard", lambda t: pytest.fail("launched"))
    a = int8.Rows(torch.zeros(8, 112, dtype=torch.int8)[:0, :K], torch.zeros(0))
    b = int8.Columns(torch.ones(3, 40, K, dtype=torch.int8).transpose(1, 2), torch.ones(3, 40))
    out = int8.grouped_int8_mm(a, b, torch.tensor([1, 2, M], dtype=torch.int32), torch.float32, torch.zeros(M, dtype=torch.int32))
    assert out.shape == (M, 40) and not out.any()
