"""Argument rules of the projection with adapters, checked on the CPU: every case must raise before anything is launched."""
import pytest
import torch

from grouped_mm_bf16_amd import _lib, lora

BF = torch.bfloat16


@pytest.fixture
def no_device_check(monkeypatch):
    monkeypatch.setattr(lora, "_require_gpu", lambda *tensors: None)


def bf(*shape):
    return torch.zeros(*shape, dtype=BF)


def args(**more):
    given = dict(x=bf(5, 32), weight=bf(32, 24), lora_a=bf(3, 32, 8), lora_b=bf(3, 8, 24), adapter=torch.zeros(5, dtype=torch.int32),
                 scale=torch.ones(3))
    given.update(more)
    return given


def test_cpu_tensors_are_refused():
    with pytest.raises(RuntimeError, match="GPU-only"):
        lora.lora_linear(**args())


@pytest.mark.parametrize("change,text", [
    (dict(x=bf(5, 32, 1)), "lora_linear takes"), (dict(weight=bf(1, 32, 24)), "lora_linear takes"), (dict(lora_a=bf(32, 8)), "lora_linear takes"),
    (dict(lora_b=bf(8, 24)), "lora_linear takes"), (dict(x=torch.zeros(5, 32)), "of one type"),
    (dict(weight=torch.zeros(32, 24, dtype=torch.float16)), "of one type"), (dict(lora_b=torch.zeros(3, 8, 24)), "of one type"),
    (dict(x=bf(5, 31)), "do not chain"), (dict(lora_a=bf(3, 31, 8)), "do not chain"), (dict(lora_b=bf(3, 9, 24)), "do not chain"),
    (dict(lora_b=bf(2, 8, 24)), "do not chain"), (dict(lora_b=bf(3, 8, 23)), "do not chain"),
    (dict(lora_a=bf(3, 32, 257), lora_b=bf(3, 257, 24)), "rank"), (dict(lora_a=bf(3, 32, 0), lora_b=bf(3, 0, 24)), "rank"),
    (dict(lora_a=bf(1023, 32, 1), lora_b=bf(1023, 1, 24)), "1022 adapters"), (dict(adapter=torch.zeros(5, dtype=torch.int64)), "adapter has to be"),
    (dict(adapter=torch.zeros(4, dtype=torch.int32)), "adapter has to be"), (dict(adapter=torch.zeros(10, dtype=torch.int32)[::2]), "adapter has to be"),
    (dict(scale=torch.ones(4)), "scale has to be"), (dict(scale=torch.ones(3, dtype=BF)), "scale has to be"),
    (dict(scale=torch.ones(3, requires_grad=True)), "scale has no gradient"), (dict(weight=bf(32, 48)[:, ::2]), "Invalid strides"),
])
def test_rules(no_device_check, change, text):
    with pytest.raises(RuntimeError, match=text):
        lora.lora_linear(**args(**change))


def test_c_entries_refuse_without_a_launch():
    lib = _lib.load()
    size, grad_size = lib.gmm_lora_workspace_bytes, lib.gmm_lora_grad_workspace_bytes
    assert size(-1, 8, 8, 8) == size(4, -1, 8, 8) == size(4, 8, 1 << 30, 8) == size(4, 8, 8, 0) == size(4, 8, 8, 257) == -1
    assert grad_size(4, 8, 8, 8, 1023) == -1 and grad_size(-1, 8, 8, 8, 3) == -1 and grad_size(1 << 29, 8, 8, 8, 3) == -1
    p = 1 << 12     # never read: every call is refused first
    ok = dict(x=p, w=p, a=p, b=p, adapter=p, out=p, T=4, K=32, N=24, R=8, L=3, xs=32, ws=(24, 1), as_=(256, 8, 1), bs=(192, 24, 1), os=24,
              dt=_lib.DT_BF16, work=p, nbytes=size(4, 32, 24, 8))

    def linear(**change):
        a = {**ok, **change}
        return lib.gmm_lora_linear(a["x"], a["w"], a["a"], a["b"], a["adapter"], None, a["out"], None, a["T"], a["K"], a["N"], a["R"], a["L"],
                                   a["xs"], *a["ws"], *a["as_"], *a["bs"], a["os"], a["dt"], a["work"], a["nbytes"], None)

    def add(**change):
        a = {**ok, **change}
        return lib.gmm_lora_add(a["x"], a["a"], a["b"], a["adapter"], None, a["out"], None, a["T"], a["K"], a["N"], a["R"], a["L"], a["xs"],
                                *a["as_"], *a["bs"], a["os"], a["dt"], a["work"], a["nbytes"], None)

    for name in ("x", "a", "b", "adapter"):
        assert linear(**{name: None}) == 1 and add(**{name: None}) == 1, name
    assert linear(w=None) == 1 and linear(out=None) == 1
    for call in (linear, add):
        assert call(T=-1) == 1 and call(R=0) == 1 and call(R=300) == 1 and call(L=1023) == 1 and call(dt=_lib.DT_F32) == 2
        assert call(xs=31) == 1 and call(os=23) == 1 and call(xs=1 << 40) == 1
        assert call(as_=(-1, 8, 1)) == 1 and call(bs=(0, 1 << 40, 1)) == 1
        assert call(work=None) == 4 and call(work=p + 4) == 4 and call(nbytes=0) == 4
        assert call(T=0, x=None) == 0
    assert linear(T=65) == 2 and linear(ws=(1 << 40, 1)) == 2 and linear(ws=(-1, 1)) == 1
    assert add(out=None) == 0          # nothing is wanted

    def grad(x=p, dy=p, low=p, u=p, da=p, db=p, T=4, xs=32, ds=24, L=3, nbytes=grad_size(4, 32, 24, 8, 3), work=p):
        return lib.gmm_lora_grad(x, dy, low, u, p, None, da, db, T, 32, 24, 8, L, xs, ds, 256, 8, 1, 192, 24, 1, _lib.DT_BF16, work, nbytes, None)

    assert grad(x=None) == grad(dy=None) == grad(low=None) == grad(u=None) == 1 and grad(xs=31) == grad(ds=23) == 1 and grad(L=1023) == 1
    assert grad(nbytes=0) == grad(work=None) == 4 and grad(da=None, db=None) == 0 and grad(L=0) == 0
