"""Argument rules of layer norm, checked on the CPU: every case must raise before anything is launched."""
import pytest
import torch

from grouped_mm_bf16_amd import _lib, norm

BF = torch.bfloat16


@pytest.fixture
def no_device_check(monkeypatch):
    monkeypatch.setattr(norm, "_require_gpu", lambda *tensors: None)


def bf(*shape):
    return torch.zeros(*shape, dtype=BF)


def test_cpu_tensors_are_refused():
    with pytest.raises(RuntimeError, match="GPU-only"):
        norm.layer_norm(bf(4, 8))


@pytest.mark.parametrize("x,weight,bias,text", [
    (torch.zeros(4, 8, dtype=torch.float64), None, None, "Unsupported dtype"),
    (torch.zeros(4, 8, dtype=torch.int32), None, None, "Unsupported dtype"),
    (torch.zeros((), dtype=BF), None, None, "at least one dimension"),
    (bf(1, 16385), None, None, "up to 16384"),
    (bf(4, 8), bf(7), None, "weight has to be a contiguous 1D"),
    (bf(4, 8), bf(16)[::2], None, "weight has to be a contiguous 1D"),
    (bf(4, 8), None, bf(1, 8), "bias has to be a contiguous 1D"),
    (bf(4, 8), torch.ones(8, dtype=torch.float16), None, "both float32"),
    (bf(4, 8), torch.ones(8), bf(8), "both float32"),
    (torch.zeros(4, 8), bf(8), None, "both float32"),
])
@pytest.mark.parametrize("graph", [False, True])
def test_rules(no_device_check, x, weight, bias, text, graph):
    if graph and x.is_floating_point():
        x = x.detach().requires_grad_()
    with pytest.raises(RuntimeError, match=text):
        norm.layer_norm(x, weight, bias)


def test_c_entries_refuse_without_a_launch():
    lib = _lib.load()
    p = 1 << 12     # never read: every call is refused first
    ok = dict(rows=4, width=8, xs=8, ys=8, dt=_lib.DT_BF16, wdt=_lib.DT_BF16)

    def call(mean=None, rstd=None, x=p, y=p, **change):
        a = {**ok, **change}
        return lib.gmm_layer_norm(x, p, p, y, mean, rstd, a["rows"], a["width"], a["xs"], a["ys"], 1e-5, a["dt"], a["wdt"], None)

    assert call(rows=-1) == 1 and call(width=-1) == 1 and call(width=16385) == 1
    assert call(x=None) == 1 and call(y=None) == 1 and call(mean=p) == 1 and call(xs=7) == 1 and call(ys=0) == 1
    assert call(dt=3) == 2 and call(dt=-1) == 2 and call(wdt=_lib.DT_F16) == 2 and call(dt=_lib.DT_F32) == 2
    assert call(rows=0, x=None) == 0 and call(width=0, y=None) == 0
    assert lib.gmm_layer_norm_workspace_bytes(-1, 8) == -1 and lib.gmm_layer_norm_workspace_bytes(4, 16385) == -1

    def back(dy=p, x=p, dx=p, dw=p, ws=None, nbytes=0, rows=4, width=8, ds=8):
        return lib.gmm_layer_norm_backward(dy, x, p, p, p, dx, dw, None, rows, width, ds, 8, 8, _lib.DT_BF16, _lib.DT_BF16, ws, nbytes, None)

    assert back(dy=None) == 1 and back(x=None) == 1 and back(ds=4) == 1 and back(width=20000) == 1
    assert back(ws=None, nbytes=1 << 30) == 4
    assert back(dx=None, dw=None) == 0 and back(width=0) == 0
