"""Argument rules of the 8-bit products, checked on the CPU: every case must raise before anything is launched; and the assembly tile on 8-bit
integers, whose waits are checked as the 16-bit tile's are."""
import pytest
import torch

import test_tile_asm_waits as waits
from grouped_mm_bf16_amd import _lib, int8, moe

BF = torch.bfloat16


@pytest.fixture
def no_launch(monkeypatch):
    """No check of devices, and no launch that is not expected."""
    def refuse(*args):
        raise AssertionError("launched")
    monkeypatch.setattr(int8, "_require_gpu", lambda *tensors: None)
    for name in ("_quantize_now", "_mm_now", "_gated_now"):
        monkeypatch.setattr(int8, name, refuse)
    monkeypatch.setattr(moe, "_route_now", refuse)


def rows(M=4, K=32, **change):
    return int8.Rows(torch.zeros(M, K, dtype=torch.int8), torch.zeros(M))._replace(**change)


def columns(*lead, K=32, N=8, **change):
    return int8.Columns(torch.zeros(*lead, N, K, dtype=torch.int8).transpose(-2, -1), torch.zeros(*lead, N))._replace(**change)


def test_cpu_tensors_are_refused():
    offs = torch.zeros(2, dtype=torch.int32)
    for call in (lambda: int8.quantize_rows(torch.zeros(4, 8)), lambda: int8.quantize_columns(torch.zeros(4, 8)), lambda: int8.int8_mm(rows(), columns()),
                 lambda: int8.grouped_int8_mm(rows(), columns(2), offs), lambda: int8.linear_int8(torch.zeros(4, 32), columns()),
                 lambda: int8.moe_forward_int8(torch.zeros(4, 32, dtype=BF), torch.zeros(4, 2), columns(2, N=16), columns(2, K=8, N=32), 1)):
        with pytest.raises(RuntimeError, match="GPU-only"):
            call()


@pytest.mark.parametrize("x,text", [(torch.zeros(4, 8, dtype=torch.float64), "Unsupported dtype"), (torch.zeros(4, 8, dtype=torch.int8), "Unsupported dtype"),
                                    (torch.zeros(4), "2D"), (torch.zeros(2, 2, 4, 4), "2D"), (torch.zeros(4, 8, requires_grad=True), "forward only")])
def test_rounding_rules(no_launch, x, text):
    for f in (int8.quantize_rows, int8.quantize_columns):
        with pytest.raises(RuntimeError, match=text):
            f(x)


def test_scales_that_require_a_gradient(no_launch, monkeypatch):
    """They would be constants without a word."""
    learned = lambda t: t._replace(scale=t.scale.clone().requires_grad_())
    offs, x, z = torch.zeros(2, dtype=torch.int32), torch.zeros(4, 32, dtype=BF), torch.zeros(4, 2)
    calls = [lambda: int8.int8_mm(learned(rows()), columns()), lambda: int8.int8_mm(rows(), learned(columns())),
             lambda: int8.grouped_int8_mm(learned(rows()), columns(2), offs), lambda: int8.grouped_int8_mm(rows(), learned(columns(2)), offs),
             lambda: int8.linear_int8(x, learned(columns())),
             lambda: int8.moe_forward_int8(x, z, learned(columns(2, N=16)), columns(2, K=8, N=32), 1),
             lambda: int8.moe_forward_int8(x, z, columns(2, N=16), learned(columns(2, K=8, N=32)), 1)]
    for call in calls:
        with pytest.raises(RuntimeError, match="forward only"):
            call()
    monkeypatch.setattr(int8, "_mm_now", lambda a, *rest: torch.ones(1))
    with torch.no_grad():
        assert calls[0]() == calls[1]() == calls[2]() == calls[3]() == 1


BAD_ROWS = [(rows(values=torch.zeros(4, 32)), "2D int8"), (rows(values=torch.zeros(32, dtype=torch.int8)), "2D int8"),
            (rows(scale=torch.zeros(3)), "rows' scale"), (rows(scale=torch.zeros(4, dtype=BF)), "rows' scale"), (rows(scale=torch.zeros(8)[::2]), "rows' scale"),
            (rows(K=31), "contraction dimensions")]


@pytest.mark.parametrize("a,text", BAD_ROWS)
def test_rows_rules(no_launch, a, text):
    with pytest.raises(RuntimeError, match=text):
        int8.int8_mm(a, columns())
    with pytest.raises(RuntimeError, match=text):
        int8.grouped_int8_mm(a, columns(2), torch.zeros(2, dtype=torch.int32))


@pytest.mark.parametrize("change,text", [
    (dict(values=torch.zeros(32, 8)), "2D int8"),
    (dict(values=torch.zeros(32, 8, dtype=torch.int8)), "contiguous along K"),
    (dict(values=torch.zeros(2, 8, 32, dtype=torch.int8).transpose(1, 2)), "2D int8"),
    (dict(scale=torch.zeros(7)), "columns' scale"),
    (dict(scale=torch.zeros(8, dtype=BF)), "columns' scale"),
    (dict(scale=torch.zeros(16)[::2]), "columns' scale"),
])
def test_columns_rules(no_launch, change, text):
    for call in (lambda b: int8.int8_mm(rows(), b), lambda b: int8.linear_int8(torch.zeros(4, 32), b)):
        with pytest.raises(RuntimeError, match=text):
            call(columns(**change))


def test_depth_rule(no_launch):
    K = int8.MAX_K + 1
    with pytest.raises(RuntimeError, match="at most 131071"):
        int8.int8_mm(rows(1, K), columns(K=K, N=1))


@pytest.mark.parametrize("offs,text", [(torch.zeros(3, dtype=torch.int32), "batch sizes"), (torch.zeros(2, dtype=torch.int64), "int32"),
                                       (torch.zeros(4, dtype=torch.int32)[::2], "int32"), (torch.zeros(2, 1, dtype=torch.int32), "int32")])
def test_group_rules(no_launch, offs, text):
    with pytest.raises(RuntimeError, match=text):
        int8.grouped_int8_mm(rows(), columns(2), offs)


@pytest.mark.parametrize("index", [torch.zeros(4, dtype=torch.int64), torch.zeros(8, dtype=torch.int32)[::2], torch.zeros(2, 2, dtype=torch.int32)])
def test_row_index_rule(no_launch, index):
    with pytest.raises(RuntimeError, match="row_index"):
        int8.grouped_int8_mm(rows(), columns(2), torch.zeros(2, dtype=torch.int32), row_index=index)


def test_other_rules(no_launch):
    with pytest.raises(RuntimeError, match="1024 groups"):
        int8.grouped_int8_mm(rows(K=1), int8.Columns(torch.zeros(1024, 1, 1, dtype=torch.int8), torch.zeros(1024, 1)), torch.zeros(1024, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="Unsupported dtype"):
        int8.int8_mm(rows(), columns(), torch.int8)
    with pytest.raises(RuntimeError, match="contraction dimensions"):
        int8.linear_int8(torch.zeros(4, 31), columns())
    with pytest.raises(RuntimeError, match="forward only"):
        int8.linear_int8(torch.zeros(4, 32, requires_grad=True), columns())
    with pytest.raises(RuntimeError, match="2D"):
        int8.linear_int8(torch.zeros(2, 4, 32), columns())


LAYER = dict(x=torch.zeros(4, 32, dtype=BF), z=torch.zeros(4, 2), up=columns(2, N=16), down=columns(2, K=8, N=32), kind="swiglu")


@pytest.mark.parametrize("change,text", [
    (dict(x=torch.zeros(5, 32, dtype=BF)), "agree on T"),
    (dict(x=torch.zeros(4, 32)), "bfloat16 or float16"),
    (dict(z=torch.zeros(4, 3)), "agree with router_logits on E"),
    (dict(kind="gelu"), "unknown activation"),
    (dict(kind="silu"), "do not chain"),
    (dict(up=columns(2, K=31, N=16)), "do not chain"),
    (dict(down=columns(2, K=8, N=31)), "do not chain"),
    (dict(up=columns(2, N=16, scale=torch.zeros(2, 15))), "columns' scale"),
    (dict(x=torch.zeros(4, 32, dtype=BF, requires_grad=True)), "forward only"),
    (dict(z=torch.zeros(4, 2, requires_grad=True)), "forward only"),
])
def test_layer_rules(no_launch, change, text):
    a = {**LAYER, **change}
    with pytest.raises(RuntimeError, match=text):
        int8.moe_forward_int8(a["x"], a["z"], a["up"], a["down"], 1, a["kind"])


def test_c_entries_refuse_without_a_launch():
    lib, p = _lib.load(), 1 << 12      # never read: every call is refused first, or has nothing to do

    def quantize(x=p, v=p, s=p, R=4, W=30, xs=30, vs=32, dt=0):
        return lib.gmm_int8_quantize(x, v, s, R, W, xs, vs, dt, None)

    assert quantize(R=-1) == quantize(R=1 << 31) == quantize(W=-1) == quantize(W=1 << 30) == quantize(x=None) == quantize(v=None) == quantize(s=None) == 1
    assert quantize(xs=29) == quantize(vs=31) == quantize(vs=16) == quantize(v=p + 8) == 1
    assert quantize(dt=3) == quantize(dt=-1) == 2 and quantize(R=0, x=None) == 0

    def gated(h=p, v=p, s=p, R=4, W=30, hs=60, vs=32, kind=1):
        return lib.gmm_int8_gated(h, v, s, R, W, hs, vs, kind, None)

    assert gated(R=-1) == gated(h=None) == gated(hs=59) == gated(vs=24) == gated(kind=2) == gated(kind=-1) == 1 and gated(R=0, h=None) == 0

    def mm(a=p, s=p, idx=None, b=p, t=p, out=p, offs=p, G=2, R=4, M=4, N=8, K=30, sa=32, sg=256, sn=32, so=8, dt=0):
        return lib.gmm_int8_mm(a, s, idx, b, t, out, offs, G, R, M, N, K, sa, sg, sn, so, dt, None, 0, None)

    assert mm(M=-1) == mm(N=1 << 31) == mm(K=-1) == mm(K=131072) == mm(R=-1) == mm(G=-1) == mm(G=1024) == mm(offs=None) == 1
    assert mm(out=None) == mm(R=5) == mm(so=7) == mm(s=None) == mm(t=None) == mm(a=None) == mm(b=None) == mm(a=p + 8) == mm(b=p + 1) == 1
    assert mm(sa=30) == mm(sg=250) == mm(sn=30) == mm(sa=16) == mm(sn=16) == mm(sa=-32) == mm(sn=-32) == mm(sg=-16) == 1
    assert mm(dt=3) == mm(dt=-1) == 2 and mm(sa=1 << 23) == mm(sn=1 << 23) == mm(so=1 << 22) == mm(idx=p, R=1 << 27) == 2
    assert mm(dt=2, so=1 << 21) == 2
    def gate_up(a=p, out=p, offs=p, G=2, R=4, M=4, N=128, K=30, sa=32, sg=4096, sn=32, so=64):
        return lib.gmm_int8_gate_up(a, p, p, p, p, out, offs, G, R, M, N, K, sa, sg, sn, so, None)

    assert gate_up(N=64) == gate_up(N=130) == gate_up(sn=1 << 22, N=1024, so=512) == 2
    assert gate_up(a=None) == gate_up(out=None) == gate_up(offs=None) == gate_up(so=63) == gate_up(K=-1) == gate_up(N=-128) == gate_up(offs=None, G=1) == 1 and gate_up(M=0) == 0
    assert mm(M=0, R=0, a=None) == mm(N=0, b=None) == mm(G=0, offs=p) == 0


# ------------------------------------------------------------------ the tile
def variants():
    return [waits.gen.Variant(0, 0, f32, tm, f16, b_nt, act) for f16, f32 in ((2, 0), (2, 1), (3, 0)) for tm in (4, 2, 1)
            for b_nt, act in ((0, 0), (1, 0), (0, 2), (0, 4), (1, 4)) if not (b_nt and tm == 4) and not (act and not f32)]


@pytest.mark.parametrize("v", variants(), ids=lambda v: f"{v.name}_{v.out_f32}_{v.f16}")
def test_the_tile_differs_in_its_instruction_alone(v):
    """Prologue and loop are those of the 16-bit tile, whose waits test_tile_asm_waits.py checks, but for the product.  (The copies of the scales come
    before them: every wait, which counts the youngest, covers them.)"""
    like = waits.gen.Variant(0, 0, 1 if v.out_f32 and not v.scaled_act else 0, v.tm, 0, v.b_nt, 2 if v.partial else 0)
    texts = []
    for variant in (v, like):
        e = waits.gen.Emit()
        waits.gen.gen_main(variant, e, "T")
        texts.append([line.replace(variant.mfma, "MFMA") for line in e.lines if not line.startswith("; ---- prologue")])
    assert texts[0] == texts[1]
    assert any(line.startswith("s_waitcnt vmcnt") for line in texts[0][:texts[0].index("s_barrier")])


@pytest.mark.parametrize("v", variants(), ids=lambda v: f"{v.name}_{v.out_f32}_{v.f16}")
def test_scales_lie_behind_all_buffers_and_registers(v):
    g = waits.gen
    assert v.stages * (v.a_stage + v.b_stage) <= g.SCALES and 4 * 32 * v.tm * g.PITCH <= g.SCALES
    e = g.gen_variant(v)
    reads = [line for line in e.lines if line.startswith("ds_read") and (f"v{g.V_RA + 2}" in line.split() or f"v{g.V_RB + 2} " in line + " ")]
    epilogue = e.lines[e.lines.index("; ---- epilogue"):]
    scaled = [line for line in epilogue if line.startswith("v_mul_f32") and 48 <= int(line.split()[2].strip("v,") if line.split()[2][0] == "v" else 0)]
    assert len(scaled) == (0 if v.partial else 2 * 4 * 8 * 2 * v.tm)
    used = {r for line in scaled for r in waits.regs(line.split()[2].rstrip(","))}
    assert not used or used == set(range(48, 80 + 2 * v.tm))
    assert len([line for line in epilogue if line.startswith("v_cvt_f32_i32")]) == len(scaled) // 2
    assert v.partial or len(reads) >= 8
