"""Argument rules of the expert layer for a few tokens, checked on the CPU: every case must raise before anything is launched."""
import pytest
import torch

from grouped_mm_bf16_amd import _lib, moe

BF = torch.bfloat16


@pytest.fixture
def no_device_check(monkeypatch):
    monkeypatch.setattr(moe, "_require_gpu", lambda *tensors: None)


def bf(*shape):
    return torch.zeros(*shape, dtype=BF)


def args(T=4, E=8, H=64, I=32, top_k=2, **more):
    given = dict(x=bf(T, H), router_logits=torch.zeros(T, E), w_up=bf(E, H, 2 * I), w_down=bf(E, I, H), top_k=top_k)
    given.update(more)
    return given


def test_cpu_tensors_are_refused():
    with pytest.raises(RuntimeError, match="GPU-only"):
        moe.moe_forward_few(**args())


@pytest.mark.parametrize("change,text", [
    (dict(x=bf(4, 64, 1)), "must agree on T"), (dict(x=bf(5, 64)), "must agree on T"), (dict(router_logits=torch.zeros(4, 9)), "agree with router_logits"),
    (dict(w_down=bf(7, 32, 64)), "agree with router_logits"), (dict(w_up=bf(64, 64)), "agree with router_logits"),
    (dict(activation="gelu"), "unknown activation"), (dict(activation="silu"), "do not chain"), (dict(w_down=bf(8, 32, 65)), "do not chain"),
    (dict(w_up=bf(8, 63, 64)), "do not chain"), (dict(w_up=bf(8, 64, 63), w_down=bf(8, 31, 64)), "even number"),
    (dict(interleaved=True), "blocks of 128"), (dict(interleaved=True, activation="silu"), "go with the swiglu"),
    (dict(x=bf(65, 64), router_logits=torch.zeros(65, 8)), "up to 64 tokens"),
    (dict(x=torch.zeros(4, 64)), "of one type"), (dict(w_up=torch.zeros(8, 64, 64, dtype=torch.float16)), "of one type"),
    (dict(router_logits=torch.zeros(4, 8, dtype=torch.float64)), "Unsupported dtype"), (dict(top_k=0), "top_k"), (dict(top_k=9), "top_k"),
])
def test_rules(no_device_check, change, text):
    with pytest.raises(RuntimeError, match=text):
        moe.moe_forward_few(**args(**change))


def test_too_many_experts(no_device_check):
    with pytest.raises(RuntimeError, match="1024 groups"):
        moe.moe_forward_few(**args(E=1024, H=1, I=1))


def test_c_entries_refuse_without_a_launch():
    lib = _lib.load()
    size = lib.gmm_moe_few_workspace_bytes
    assert size(65, 8, 2, 64, 32) == -1 and size(-1, 8, 2, 64, 32) == -1 and size(4, 8, 9, 64, 32) == -1 and size(4, 1024, 2, 64, 32) == -1
    assert size(4, 8, 2, -1, 32) == -1 and size(4, 8, 2, 64, 1 << 30) == -1 and size(0, 8, 2, 64, 32) >= 0
    need = size(4, 8, 2, 64, 32)
    p = 1 << 12     # never read: every call is refused first
    ok = dict(x=p, logits=p, up=p, down=p, out=p, T=4, E=8, k=2, H=64, I=32, xs=64, us=(64 * 64, 64, 1), ds=(32 * 64, 64, 1), os=64, kind=1,
              dt=_lib.DT_BF16, ws=p, nbytes=need)

    def call(**change):
        a = {**ok, **change}
        return lib.gmm_moe_few(a["x"], a["logits"], a["up"], a["down"], a["out"], a["T"], a["E"], a["k"], a["H"], a["I"], a["xs"], 8, *a["us"],
                               *a["ds"], a["os"], a["kind"], 1, a["dt"], _lib.DT_F32, a["ws"], a["nbytes"], None)

    for name in ("x", "logits", "up", "down", "out"):
        assert call(**{name: None}) == 1, name
    assert call(T=65) == 1 and call(k=9) == 1 and call(kind=3) == 1 and call(kind=-1) == 1 and call(kind=2) == 1 and call(dt=_lib.DT_F32) == 2
    assert call(xs=63) == 1 and call(os=63) == 1 and call(xs=1 << 40) == 1 and call(us=(-1, 64, 1)) == 1
    assert call(us=(0, 1 << 40, 1)) == 1 and call(ds=(0, 64, -1)) == 1                 # 2 GiB and more, negative
    assert call(nbytes=need - 1) == 4 and call(ws=None) == 4 and call(ws=p + 4) == 4
    assert call(T=0, x=None) == 0
