"""Refusals of gmm_moe_sum_rows_f32, gmm_moe_route and gmm_moe_route_own through the C interface: every call is refused before a launch, or has nothing to do."""
import pytest

from grouped_mm_bf16_amd import _lib

P = 1 << 12      # never read


def test_sums_of_rows_in_fp32():
    lib = _lib.load()

    def total(y=P, rows=P, w=P, out=P, T=4, k=2, H=8, R=8, ys=8, os=8, dt=0):
        return lib.gmm_moe_sum_rows_f32(y, rows, w, out, T, k, H, R, ys, os, dt, None)

    assert total(T=-1) == total(T=1 << 31) == total(k=0) == total(k=33) == total(H=-1) == total(R=-1) == 1
    assert total(y=None) == total(rows=None) == total(out=None) == total(ys=7) == total(os=7) == 1
    assert total(dt=3) == total(dt=-1) == 2
    assert total(T=0, y=None) == total(H=0, y=None) == 0


@pytest.mark.parametrize("name", ["gmm_moe_route", "gmm_moe_route_own"])
def test_routing(name):
    lib = _lib.load()

    def route(z=P, ld=8, dt=2, T=4, E=8, k=2, offs=P, expert=P, weight=P, token=P, rows=P, ws=P, size=1 << 20):
        return getattr(lib, name)(z, ld, dt, T, E, k, 1, offs, expert, weight, token, rows, ws, size, None)

    assert route(T=-1) == route(E=0) == route(E=1024) == route(k=0) == route(k=9) == route(k=33, E=40) == route(size=-1) == 1
    assert route(z=None) == route(offs=None) == route(expert=None) == route(weight=None) == route(token=None) == route(rows=None) == route(ws=None) == 1
    assert route(ld=7) == 1 and route(dt=3) == 2 and route(size=31) == _lib.ERR_WORKSPACE
    assert route(T=1 << 30) == 1      # 2^31 slots
