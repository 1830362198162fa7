"""The workspace of a routing call through the C interface, on a real MI355X: left alone up to 131072 slots, so that calls on several streams may share one, and used
from gmm_moe_route_own's first counted slot on by the call that has one of its own."""
import pytest
import torch

from grouped_mm_bf16_amd import _lib

pytestmark = pytest.mark.gpu
DEV = "cuda"


def call(entry, logits, k, ws, stream):
    T, E = logits.shape
    ints = lambda n: torch.full((n,), -7, dtype=torch.int32, device=DEV)
    held = [ints(E), ints(T * k), torch.empty(T * k, device=DEV), ints(T * k), ints(T * k)]
    rc = entry(logits.data_ptr(), E, _lib.DT_F32, T, E, k, 1, *(t.data_ptr() for t in held), ws.data_ptr(), 4 * ws.numel(), stream)
    assert rc == _lib.OK
    return held


def logits_of(T, E, seed=0):
    return torch.randn(T, E, device=DEV, generator=torch.Generator(device=DEV).manual_seed(T + E + seed))


def check(held, k):
    offs, expert, _, row_token, token_rows = held
    order = torch.sort(expert.long(), stable=True).indices
    want = torch.empty_like(order)
    want[order] = torch.arange(order.numel(), device=DEV)
    assert torch.equal(row_token.long(), order // k) and torch.equal(token_rows.long(), want)
    assert torch.equal(offs.long(), torch.bincount(expert.long(), minlength=offs.numel()).cumsum(0))


@pytest.mark.parametrize("T,E,k", [(100, 8, 2), (2048, 128, 8), (16385, 8, 1), (3000, 60, 7), (16384, 128, 8), (65536, 3, 2), (131072, 4, 1), (4096, 1023, 32)])
def test_left_alone(T, E, k):
    lib = _lib.load()
    ws = torch.full((lib.gmm_moe_route_workspace_bytes(T, E, k) // 4,), 0x5a5a5a5a, dtype=torch.int32, device=DEV)
    held = call(lib.gmm_moe_route, logits_of(T, E), k, ws, torch.cuda.current_stream().cuda_stream)
    assert (ws == 0x5a5a5a5a).all()
    check(held, k)


@pytest.mark.parametrize("T,E,k", [(131073, 2, 1), (131072, 7, 2), (300000, 64, 1)])
def test_past_the_limit(T, E, k):
    lib = _lib.load()
    ws = torch.empty(lib.gmm_moe_route_workspace_bytes(T, E, k) // 4, dtype=torch.int32, device=DEV)
    check(call(lib.gmm_moe_route, logits_of(T, E), k, ws, torch.cuda.current_stream().cuda_stream), k)


def test_shared_by_two_streams():
    lib = _lib.load()
    logits = [logits_of(16384, 64, seed) for seed in (0, 1)]
    ws = torch.empty(lib.gmm_moe_route_workspace_bytes(16384, 64, 8) // 4, dtype=torch.int32, device=DEV)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, (s, t) in enumerate(zip(streams, logits)):
            with torch.cuda.stream(s):
                got[i].append(call(lib.gmm_moe_route, t, 8, ws, s.cuda_stream))
    torch.cuda.synchronize()
    for calls in got:
        check(calls[0], 8)
        assert all(torch.equal(p, q) for other in calls[1:] for p, q in zip(calls[0], other))


@pytest.mark.parametrize("T,E,k", [(5, 8, 2), (16384, 64, 1), (16385, 64, 1), (16384, 128, 8), (131073, 2, 1), (300000, 4, 1)])
def test_of_ones_own(T, E, k):
    """The same results, on a workspace with anything in it."""
    lib = _lib.load()
    ws = torch.full((lib.gmm_moe_route_workspace_bytes(T, E, k) // 4,), -1, dtype=torch.int32, device=DEV)
    stream = torch.cuda.current_stream().cuda_stream
    own = call(lib.gmm_moe_route_own, logits_of(T, E), k, ws, stream)
    check(own, k)
    assert all(torch.equal(p, q) for p, q in zip(own, call(lib.gmm_moe_route, logits_of(T, E), k, ws, stream)))
    assert lib.gmm_moe_route_own(logits_of(T, E).data_ptr(), E, _lib.DT_F32, T, E, k, 1, *(t.data_ptr() for t in own), ws.data_ptr(), 4 * ws.numel() - 4, stream) == _lib.ERR_WORKSPACE
