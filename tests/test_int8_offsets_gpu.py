"""Offsets of 8-bit grouped products that go down as well as up, on a real MI355X, where rows are few enough to be streamed and where they are not: group g is
offs[g - 1] .. offs[g] - 1, clamped to the rows there are, a row that one group alone claims is that group's, each element of one that several claim is one of theirs."""
import pytest
import torch

from grouped_mm_bf16_amd import int8
from oracle import int8_oracle as oracle

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = torch.bfloat16


def check(M, offs, gather, K=64, N=72):
    G = len(offs)
    gen = torch.Generator().manual_seed(M + G + K)
    values = lambda *shape: torch.randint(-128, 128, shape, generator=gen, dtype=torch.int8).to(DEV)
    a = int8.Rows(values(M, K), 1e-2 + torch.rand(M, generator=gen).to(DEV))
    b = int8.Columns(values(G, N, K).transpose(1, 2), 1e-2 + torch.rand(G, N, generator=gen).to(DEV))
    index = torch.randperm(M, generator=gen).to(torch.int32).to(DEV) if gather else None
    rows = a if index is None else int8.Rows(a.values[index.long()], a.scale[index.long()])
    torch.full((M * N,), float("nan"), dtype=BF, device=DEV)      # what an allocation finds, where it finds it again
    out = int8.grouped_int8_mm(a, b, torch.tensor(offs, dtype=torch.int32, device=DEV), BF, index).double().cpu()
    ends = [0] + [min(max(end, 0), M) for end in offs]
    fits, claims = torch.zeros(M, N, dtype=torch.bool), torch.zeros(M, dtype=torch.int32)
    for g, (first, end) in enumerate(zip(ends, ends[1:])):
        if end > first:
            want, bound = oracle.mm(rows.values[first:end], rows.scale[first:end], b.values[g], b.scale[g], BF)
            fits[first:end] |= (out[first:end] - want).abs() <= bound
            claims[first:end] += 1
    wrong = (claims > 0) & ~fits.all(1)
    assert not wrong.any(), f"{M} rows, {offs[:12]}: {wrong.nonzero()[:, 0].tolist()} are no group's that claims them"


OFFSETS = [(100, [90, 0, 90, 0, 90, 0, 90, 100]), (4, [1, 0, 1, 0, 1, 0, 1, 4]), (5, [3, 1, 3, 1, 3, 5, 2, 5, 0]), (64, [60, 0, 60, 0, 60, 64]), (64, [64, 0, 64, 0, 64, 0, 64]),
           (40, [40, -3, 7, 5, 99, 2, 40]), (1, [1, 0, 1, 0, 1]), (3, [0, 0, 2, 0, 3]), (200, [33, 1, 65, 2, 97, 3, 200, 199, 200, 5])]


@pytest.mark.parametrize("gather", [False, True])
@pytest.mark.parametrize("M,offs", OFFSETS)
def test_up_and_down(M, offs, gather):
    check(M, offs, gather)
    check(M, offs, gather, K=67)      # an odd one: through tiles


@pytest.mark.parametrize("M,G", [(4, 100), (30, 70), (64, 129), (256, 200), (1000, 300), (1024, 1023)])
def test_at_random(M, G):
    """More groups than a wave looks at together; every second one below the one before."""
    gen = torch.Generator().manual_seed(M * G)
    for most in (M, M + 50):
        offs = torch.randint(-5, most + 1, (G,), generator=gen)
        offs[-1] = M
        check(M, offs.tolist(), False, K=32, N=24)
    up = torch.randint(0, M + 1, (G,), generator=gen).sort().values
    up[G // 3], up[G // 2] = 0, M
    check(M, up.tolist(), True, K=32, N=24)
