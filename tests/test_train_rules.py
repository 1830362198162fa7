"""Argument rules of the steps of an expert layer that is trained and of dropout, checked on the CPU: every case must raise before anything is
launched; derivatives that there are not raise (the kernels are replaced by the formulas)."""
import pytest
import torch
from torch.autograd import forward_ad

from grouped_mm_bf16_amd import _lib, dropout, moe, moe_train

BF = torch.bfloat16


@pytest.fixture
def no_device_check(monkeypatch):
    for module in (moe_train, dropout, moe):
        monkeypatch.setattr(module, "_require_gpu", lambda *tensors: None)


def routing(tokens=4, k=2, **change):
    slots = tokens * k
    ints = lambda n: torch.zeros(n, dtype=torch.int32)
    r = moe.Routing(ints(3), ints(slots), torch.zeros(slots), ints(slots), torch.arange(slots, dtype=torch.int32))
    return r._replace(**change)


def test_cpu_tensors_are_refused():
    for call in (lambda: moe_train.sort_rows(torch.zeros(4, 8), routing()), lambda: moe_train.combine_rows(torch.zeros(8, 8), routing(), 2),
                 lambda: moe_train.gated(torch.zeros(4, 8)), lambda: moe_train.route(torch.zeros(4, 8), 2),
                 lambda: dropout.dropout(torch.zeros(4), 0.5, torch.zeros(2, dtype=torch.int64))):
        with pytest.raises(RuntimeError, match="GPU-only"):
            call()


@pytest.mark.parametrize("x,change,text", [
    (torch.zeros(4, 8, dtype=torch.float64), {}, "Unsupported dtype"),
    (torch.zeros(4), {}, "2D"),
    (torch.zeros(2, 4, 8), {}, "2D"),
    (torch.zeros(3, 8), {}, "has to have"),
    (torch.zeros(9, 8), {}, "top_k|has to have"),
    (torch.zeros(4, 8), {"token_rows": torch.zeros(8, dtype=torch.int64)}, "contiguous 1D torch.int32"),
    (torch.zeros(4, 8), {"token_rows": torch.zeros(16, dtype=torch.int32)[::2]}, "contiguous 1D torch.int32"),
    (torch.zeros(4, 8), {"token_rows": torch.zeros(8, 1, dtype=torch.int32)}, "contiguous 1D torch.int32"),
    (torch.zeros(4, 8), {"token_rows": torch.zeros(132, dtype=torch.int32)}, "top_k has to be in"),
])
@pytest.mark.parametrize("graph", [False, True])
def test_sort_rules(no_device_check, x, change, text, graph):
    with pytest.raises(RuntimeError, match=text):
        moe_train.sort_rows(x.detach().requires_grad_(graph), routing(**change))


@pytest.mark.parametrize("y,k,change,text", [
    (torch.zeros(8, 8, dtype=torch.int32), 2, {}, "Unsupported dtype"),
    (torch.zeros(8), 2, {}, "2D"),
    (torch.zeros(8, 8), 0, {}, "top_k has to be in"),
    (torch.zeros(8, 8), 33, {}, "top_k has to be in"),
    (torch.zeros(8, 8), 3, {}, "tokens \\* top_k rows"),
    (torch.zeros(7, 8), 2, {}, "has to have"),
    (torch.zeros(8, 8), 2, {"slot_weight": torch.zeros(8, dtype=BF)}, "slot_weight has to be a contiguous 1D torch.float32"),
    (torch.zeros(8, 8), 2, {"slot_weight": torch.zeros(4)}, "slot_weight has to have"),
    (torch.zeros(8, 8), 2, {"token_rows": torch.zeros(4, dtype=torch.int32)}, "token_rows has to have"),
])
def test_combine_rules(no_device_check, y, k, change, text):
    with pytest.raises(RuntimeError, match=text):
        moe_train.combine_rows(y, routing(**change), k)


@pytest.mark.parametrize("h,kind,text", [
    (torch.zeros(4, 8, dtype=torch.float64), "swiglu", "Unsupported dtype"),
    (torch.zeros(8), "swiglu", "2D"),
    (torch.zeros(4, 7), "swiglu", "even number"),
    (torch.zeros(4, 8), "gelu", "unknown activation"),
])
def test_activation_rules(no_device_check, h, kind, text):
    with pytest.raises(RuntimeError, match=text):
        moe_train.gated(h, kind)


@pytest.mark.parametrize("shapes,text", [
    (((4, 8), (5, 3), (3, 8, 8), (3, 4, 8)), "agree on T"),
    (((4, 8), (4, 2), (3, 8, 8), (3, 4, 8)), "agree with router_logits on E"),
    (((4, 8), (4, 3), (3, 7, 8), (3, 4, 8)), "do not chain"),
    (((4, 8), (4, 3), (3, 8, 8), (3, 8, 8)), "do not chain"),
])
def test_layer_rules(no_device_check, shapes, text):
    with pytest.raises(RuntimeError, match=text):
        moe_train.moe_train(*(torch.zeros(s) for s in shapes), 2)


def state(*shape, dtype=torch.int64):
    return torch.zeros(*shape or (2,), dtype=dtype)


@pytest.mark.parametrize("args,text", [
    ((torch.zeros(4, dtype=torch.float64), 0.5, state()), "Unsupported dtype"),
    ((torch.zeros(4), -0.1, state()), "p has to be in"),
    ((torch.zeros(4), 1.1, state()), "p has to be in"),
    ((torch.zeros(4), float("nan"), state()), "p has to be in"),
    ((torch.zeros(4), 0.5, state(3)), "rng has to be"),
    ((torch.zeros(4), 0.5, state(2, dtype=torch.int32)), "rng has to be"),
    ((torch.zeros(4), 0.5, state(4)[::2]), "rng has to be"),
    ((torch.zeros(4), 0.5, state(), torch.zeros(1, 4)), "residual has to be"),
    ((torch.zeros(4), 0.5, state(), torch.zeros(4, dtype=BF)), "residual has to be"),
    ((torch.zeros(4), 0.5, state(), None, -1), "site has to be"),
    ((torch.zeros(4), 0.5, state(), None, 65536), "site has to be"),
])
def test_dropout_rules(no_device_check, args, text):
    with pytest.raises(RuntimeError, match=text):
        dropout.dropout(*args)


# ------------------------------------------------------------------ C entries
def test_c_entries_refuse_without_a_launch():
    lib, p = _lib.load(), 1 << 12      # never read: every call is refused first, or has nothing to do

    def sort(x=p, rows=p, out=p, T=4, k=2, H=8, R=8, xs=8, os=8, dt=0):
        return lib.gmm_moe_sort_rows(x, rows, out, T, k, H, R, xs, os, dt, None)

    assert sort(T=-1) == sort(T=1 << 31) == sort(k=0) == sort(k=33) == sort(H=-1) == sort(H=1 << 31) == sort(R=-1) == 1
    assert sort(x=None) == sort(rows=None) == sort(out=None) == sort(xs=7) == sort(os=7) == 1
    assert sort(dt=3) == sort(dt=-1) == 2
    assert sort(T=0, x=None) == sort(H=0, out=None) == sort(R=0, out=None) == 0

    def total(y=p, rows=p, w=p, out=p, T=4, k=2, H=8, R=8, ys=8, os=8, dt=0):
        return lib.gmm_moe_sum_rows(y, rows, w, out, T, k, H, R, ys, os, dt, None)

    assert total(T=-1) == total(k=33) == total(y=None) == total(rows=None) == total(out=None) == total(ys=7) == total(os=7) == 1
    assert total(dt=9) == 2 and total(T=0, y=None) == total(H=0, y=None) == 0

    def back(d=p, y=p, rows=p, w=p, dy=p, dw=p, T=4, k=2, H=8, R=8, ds=8, ys=8, dys=8, dt=0):
        return lib.gmm_moe_combine_backward(d, y, rows, w, dy, dw, T, k, H, R, ds, ys, dys, dt, None)

    assert back(T=-1) == back(k=0) == back(d=None) == back(y=None) == back(rows=None) == back(w=None) == back(ds=7) == back(ys=7) == back(dys=7) == 1
    assert back(dt=3) == 2 and back(T=0) == back(dy=None, dw=None, d=None) == 0

    def route(dw=p, e=p, w=p, z=None, dl=p, T=4, E=8, k=2, zs=8, dt=0):
        return lib.gmm_moe_route_backward(dw, e, w, z, dl, T, E, k, zs, dt, None)

    assert route(T=-1) == route(E=0) == route(E=1024) == route(k=0) == route(k=9) == route(k=33, E=40) == 1
    assert route(dw=None) == route(e=None) == route(w=None) == route(dl=None) == route(z=p, zs=7) == 1
    assert route(dt=3) == 2 and route(T=0, dw=None) == 0

    def gated(h=p, out=p, rows=4, inner=8, hs=16, os=8, kind=1, dt=0):
        return lib.gmm_gated(h, out, rows, inner, hs, os, kind, dt, None)

    assert gated(rows=-1) == gated(inner=-1) == gated(inner=1 << 31) == gated(kind=2) == gated(kind=-1) == gated(h=None) == gated(out=None) == 1
    assert gated(hs=15) == gated(os=7) == 1 and gated(dt=3) == 2 and gated(rows=0, h=None) == gated(inner=0, h=None) == 0

    def gated_back(d=p, h=p, dh=p, rows=4, inner=8, ds=8, hs=16, dhs=16, kind=1, dt=0):
        return lib.gmm_gated_backward(d, h, dh, rows, inner, ds, hs, dhs, kind, dt, None)

    assert gated_back(d=None) == gated_back(h=None) == gated_back(dh=None) == gated_back(ds=7) == gated_back(hs=15) == gated_back(dhs=15) == 1
    assert gated_back(rows=0, d=None) == 0

    def drop(x=p, res=p, out=p, rng=p, used=None, rows=4, width=8, xs=8, rs=8, os=8, limit=100, site=0, dt=0):
        return lib.gmm_dropout(x, res, out, rng, used, rows, width, xs, rs, os, limit, site, dt, None)

    assert drop(rows=-1) == drop(width=-1) == drop(limit=-1) == drop(limit=65537) == drop(site=-1) == drop(site=65536) == 1
    assert drop(rows=1 << 30, width=1 << 30, xs=1 << 30, rs=1 << 30, os=1 << 30) == 1
    assert drop(x=None) == drop(out=None) == drop(rng=None) == drop(xs=7) == drop(rs=7) == drop(os=7) == 1
    assert drop(dt=3) == 2 and drop(rows=0, x=None) == drop(width=0, x=None) == 0


# ------------------------------------------------------------------ derivatives
@pytest.fixture
def formulas(no_device_check, monkeypatch):
    """The launches, as opaque to torch as they are."""
    def opaque(f):
        def g(*args):
            with torch.no_grad():
                return f(*args)
        return g

    def slots(rows, tokens):
        return rows.long().reshape(tokens, -1)

    def total(y, rows, w, tokens, k):
        terms = y[slots(rows, tokens)]
        return (terms if w is None else terms * w.reshape(tokens, -1, 1)).sum(1)

    def combine_back(grad, y, rows, w, k, need_y, need_w):
        at = slots(rows, grad.size(0))
        dy = torch.zeros(at.numel(), grad.size(1))
        dy[at.reshape(-1)] = (grad[:, None] * w.reshape(-1, k, 1)).reshape(at.numel(), -1)
        return [dy, (y[at] * grad[:, None]).sum(2).reshape(-1) if need_w else None]

    def sort(x, rows):
        out = torch.zeros(rows.numel(), x.size(1))
        out[rows.long()] = x.repeat_interleave(rows.numel() // x.size(0), 0)
        return out

    def gated(h, kind):
        return torch.nn.functional.silu(h[:, :4]) * h[:, 4:]

    def gated_back(grad, h, kind):
        with torch.enable_grad():
            leaf = h.detach().requires_grad_()
            return torch.autograd.grad(gated(leaf, kind), leaf, grad)[0]

    keep = (torch.arange(24).reshape(3, 8) % 3 > 0).float() * 1.5
    for module, name, to in ((moe_train, "_sort_now", sort), (moe_train, "_sum_now", total), (moe_train, "_combine_backward_now", combine_back),
                             (moe_train, "_gated_now", gated), (moe_train, "_gated_backward_now", gated_back),
                             (moe_train, "_route_backward_now", lambda dw, e, w, z, T, E, k, dt: torch.ones(T, E)),
                             (moe, "_route_now", lambda z, k, r: torch.zeros(z.size(1) + 4 * z.size(0) * k, dtype=torch.int32)),
                             (dropout, "_forward_now", lambda x, limit, rng, site, res: (x * keep + (0 if res is None else res), rng.clone())),
                             (dropout, "_launch", lambda x, *rest: x * keep), (dropout, "_backward_now", lambda g, *rest: g * keep)):
        monkeypatch.setattr(module, name, opaque(to))


def calls():
    order = torch.tensor([3, 0, 5, 2, 1, 4], dtype=torch.int32)
    gen = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=gen)
    two = routing(3, 2, token_rows=order)
    return {
        "sort_rows": (lambda x: moe_train.sort_rows(x, two), [r(3, 8)]),
        "combine_rows": (lambda y, w: moe_train.combine_rows(y, two._replace(slot_weight=w), 2), [r(6, 8), r(6)]),
        "gated": (lambda h: moe_train.gated(h), [r(3, 8)]),
        "route": (lambda z: moe_train.route(z, 2).slot_weight, [r(3, 4)]),
        "dropout": (lambda x, res: dropout.dropout(x, 0.3, torch.zeros(2, dtype=torch.int64), res), [r(3, 8), r(3, 8)]),
    }


NAMES = pytest.mark.parametrize("name", ["sort_rows", "combine_rows", "gated", "route", "dropout"])


@NAMES
def test_first_derivatives(formulas, name):
    """Each operand's alone and all together, with and without create_graph."""
    f, leaves = calls()[name]
    for which in [*range(len(leaves)), None]:
        mine = [t.detach().requires_grad_(which in (i, None)) for i, t in enumerate(leaves)]
        y = f(*mine)
        need = [t for t in mine if t.requires_grad]
        grads = torch.autograd.grad(y, need, torch.ones_like(y), retain_graph=True)
        again = torch.autograd.grad(y, need, torch.ones_like(y), create_graph=True)
        for p, q, t in zip(grads, again, need):
            assert p.shape == t.shape and torch.equal(p, q.detach())
    assert not f(*(t.detach() for t in leaves)).requires_grad
    with torch.no_grad():
        assert not f(*mine).requires_grad


@NAMES
def test_second_derivatives_raise(formulas, name):
    f, leaves = calls()[name]
    for which in range(len(leaves)):
        mine = [t.detach().requires_grad_(i == which) for i, t in enumerate(leaves)]
        y = f(*mine)
        value = (y ** 3).sum()
        grad, = torch.autograd.grad(value, mine[which], create_graph=True)
        if name == "dropout" and which == 1:
            continue      # the residual's gradient is the upstream one, whose derivative torch has
        with pytest.raises(RuntimeError, match="no second derivative"):
            (value + grad.square().sum()).backward()


@NAMES
def test_forward_mode_raises(formulas, name):
    f, leaves = calls()[name]
    with forward_ad.dual_level():
        f(*leaves)       # no tangent: as ever
        leaves[0] = forward_ad.make_dual(leaves[0], torch.ones_like(leaves[0]))
        with pytest.raises(NotImplementedError, match="jvp"):
            f(*leaves)
