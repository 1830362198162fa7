"""Routing and sorting of so many slots that their counts come from a kernel of their own, on a real MI355X: the sort against torch's stable one, and
against the routing that has no table of its own, around every size where another kernel takes over."""
import pytest
import torch

from grouped_mm_bf16_amd import _lib, moe

pytestmark = pytest.mark.gpu
DEV = "cuda"


def check(logits, k):
    T, E = logits.shape
    r = moe.moe_route(logits, k)
    order = torch.sort(r.slot_expert.long(), stable=True).indices
    assert torch.equal(r.row_token.long(), order // k)
    want = torch.empty_like(order)
    want[order] = torch.arange(order.numel(), device=DEV)
    assert torch.equal(r.token_rows.long(), want)
    assert torch.equal(r.offs.long(), torch.bincount(r.slot_expert.long(), minlength=E).cumsum(0))
    return r


SIZES = [(8192, 8, 2), (8193, 8, 2), (16385, 1, 1), (2049, 128, 8), (3000, 60, 7), (2500, 1000, 9), (4100, 1023, 16), (16384, 64, 8), (16385, 64, 8), (32768, 3, 3),
         (65536, 4, 4), (65537, 4, 4), (32769, 20, 8), (262144, 2, 1), (262145, 2, 1), (5000, 257, 32)]


@pytest.mark.parametrize("T,E,k", SIZES)
def test_random_choices(T, E, k):
    check(torch.randn(T, E, device=DEV, generator=torch.Generator(device=DEV).manual_seed(T + E)), k)


@pytest.mark.parametrize("T", [20000, 131000, 200001])
@pytest.mark.parametrize("expert", [0, 5, 6])
def test_all_on_one_expert(T, expert):
    logits = torch.zeros(T, 7, device=DEV)
    logits[:, expert] = 1
    check(logits, 1)


@pytest.mark.parametrize("T,E,k", [(20000, 8, 1), (3000, 128, 8), (40000, 16, 4)])
def test_as_without_a_table_and_replayed(T, E, k):
    logits = torch.randn(T, E, device=DEV, generator=torch.Generator(device=DEV).manual_seed(T))
    r = check(logits, k)
    S, lib = T * k, _lib.load()
    ints = lambda n: torch.empty(n, dtype=torch.int32, device=DEV)
    other = [ints(E), ints(S), torch.empty(S, device=DEV), ints(S), ints(S)]
    stream = torch.cuda.current_stream().cuda_stream
    rc = lib.gmm_moe_route_noalloc(logits.data_ptr(), E, _lib.DT_F32, T, E, k, 1, *(t.data_ptr() for t in other), stream)
    assert rc == 0 and all(torch.equal(p, q) for p, q in zip(r, other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = moe.moe_route(logits, k)
    for seed in range(3):
        logits.copy_(torch.randn(T, E, device=DEV, generator=torch.Generator(device=DEV).manual_seed(seed)))
        want = check(logits, k)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(held, want))


def test_on_two_streams_at_once():
    a, b = (torch.randn(16384, 64, device=DEV, generator=torch.Generator(device=DEV).manual_seed(s)) for s in (0, 1))
    want = [check(t, 4) for t in (a, b)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, (s, t) in enumerate(zip(streams, (a, b))):
            with torch.cuda.stream(s):
                got[i].append(moe.moe_route(t, 4))
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for i in range(2) for r in got[i] for p, q in zip(r, want[i]))
