"""The expert layer for a few tokens on a real MI355X against the formula in 64 bits: numbers of tokens around the kernels' sixteens of
rows, sizes with and without alignment, every layout of the weights, routing with experts that nobody chooses, masked or infinite
logits, values that are not finite."""
import pytest
import torch

from grouped_mm_bf16_amd import moe
from oracle import operators_oracle as oracle

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF = torch.bfloat16, torch.float16


def matrix(gen, shape, dtype, scale, lay):
    """lay: rows, cols (contiguous along k), padded (rows further apart), any (no dimension contiguous, odd address)."""
    if lay == "cols":
        return matrix(gen, (shape[0], shape[2], shape[1]), dtype, scale, "rows").transpose(1, 2)
    if lay == "any":
        wide = (torch.randn(shape[0], shape[1], 2 * shape[2] + 1, generator=gen) * scale).to(dtype).to(DEV)
        return wide[..., 1::2]
    pad = 8 if lay == "padded" else 0
    return (torch.randn(shape[0], shape[1], shape[2] + pad, generator=gen) * scale).to(dtype).to(DEV)[..., :shape[2]]


def make(T, E, H, I, kind="swiglu", lay="rows", dtype=BF, logits=torch.float32, seed=0):
    gen = torch.Generator().manual_seed(seed + T + E + H + I)
    x = torch.randn(T, H, generator=gen).to(dtype).to(DEV)
    z = torch.randn(T, E, generator=gen).to(logits).to(DEV)
    up = matrix(gen, (E, H, I if kind == "silu" else 2 * I), dtype, H ** -0.5, lay)
    down = matrix(gen, (E, I, H), dtype, max(I, 1) ** -0.5, lay)
    return x, z, up, down


def run(x, z, up, down, k, kind, renormalize=True):
    return moe.moe_forward_few(x, z, up, down, k, activation="silu" if kind == "silu" else "swiglu", renormalize=renormalize,
                               interleaved=kind == "interleaved")


def check(x, z, up, down, k, kind, renormalize=True):
    got = run(x, z, up, down, k, kind, renormalize)
    assert got.dtype == x.dtype and got.shape == x.shape
    want, bound = oracle.moe_layer(x, z.cpu(), up.cpu(), down.cpu(), k, kind, renormalize)
    oracle.assert_within(got, want, bound)
    assert torch.equal(got, run(x, z, up, down, k, kind, renormalize)), "not the same twice"
    return got


@pytest.mark.parametrize("T", [1, 2, 3, 15, 16, 17, 31, 32, 33, 48, 49, 63, 64])
@pytest.mark.parametrize("E,k", [(4, 2), (40, 6)])
def test_numbers_of_tokens(T, E, k):
    check(*make(T, E, 256, 192), k, "swiglu")


@pytest.mark.parametrize("T", [16, 17, 64])
def test_all_rows_to_one_expert(T):
    x, z, up, down = make(T, 8, 256, 192)
    z[:, 3] += 100
    check(x, z, up, down, 1, "swiglu")
    check(x, z, up, down, 8, "swiglu")


@pytest.mark.parametrize("kind", ["silu", "swiglu", "interleaved"])
@pytest.mark.parametrize("lay", ["rows", "cols", "padded", "any"])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("T", [1, 20, 40])
def test_layouts_and_kinds(kind, lay, dtype, T):
    check(*make(T, 6, 320, 192, kind, lay, dtype), 3, kind)


@pytest.mark.parametrize("H,I", [(8, 8), (1, 1), (7, 5), (129, 64), (64, 129), (40, 1000), (1000, 40), (256, 136), (264, 2056), (2056, 264),
                                 (1031, 519), (4096, 64), (64, 4096), (31, 2048)])
@pytest.mark.parametrize("lay", ["rows", "cols"])
def test_sizes(H, I, lay):
    for kind in ("silu", "swiglu"):
        check(*make(5, 7, H, I, kind, lay), 2, kind)


@pytest.mark.parametrize("E,k", [(1, 1), (64, 1), (65, 32), (128, 8), (200, 3), (1023, 2)])
@pytest.mark.parametrize("logits", [torch.float32, BF, HF])
def test_experts_and_choices(E, k, logits):
    for renormalize in (True, False):
        check(*make(9, E, 64, 64, logits=logits), k, "swiglu", renormalize)


def test_masked_and_infinite_logits():
    x, z, up, down = make(6, 10, 128, 64)
    z[0, 2:] = -float("inf")          # fewer experts left than choices
    z[1] = -float("inf")              # none left
    z[2, 4] = float("inf")
    z[3] = torch.finfo(torch.float32).min
    check(x, z, up, down, 3, "swiglu")


def test_what_nobody_chose_is_not_read():
    x, z, up, down = make(3, 12, 128, 64)
    z[:, 5:] = -1e4
    want = run(x, z, up, down, 4, "swiglu")
    up[5:], down[5:] = float("nan"), float("inf")
    assert torch.equal(run(x, z, up, down, 4, "swiglu"), want)


def test_a_token_that_is_not_finite_stays_alone():
    x, z, up, down = make(20, 4, 128, 64)
    want = run(x, z, up, down, 2, "swiglu")
    x[7, 3] = float("nan")
    got = run(x, z, up, down, 2, "swiglu")
    keep = [t for t in range(20) if t != 7]
    assert got[7].isnan().all() and torch.equal(got[keep], want[keep])


def test_activations_past_the_range_of_half_precision():
    """The activations are held as two fp16 values: one that fp16 cannot hold becomes infinite, as in moe_forward, never NaN."""
    x = torch.full((1, 64), 60.0, dtype=HF, device=DEV)
    up = torch.full((1, 64, 128), 1.0, dtype=HF, device=DEV)      # gate and partner 3840: the activation is 1.5e7
    down = torch.full((1, 64, 64), 2.0 ** -14, dtype=HF, device=DEV)
    got = run(x, torch.zeros(1, 1, device=DEV), up, down, 1, "swiglu")
    assert torch.isinf(got).all() and (got > 0).all()


@pytest.mark.parametrize("pad,offset", [(8, 0), (3, 0), (0, 1)])
def test_rows_of_x_and_logits_that_lie_apart(pad, offset):
    x, z, up, down = make(18, 6, 256, 128)
    want = run(x, z, up, down, 2, "swiglu")
    wide = torch.zeros(18, 256 + pad + offset, dtype=BF, device=DEV)
    wide[:, offset:offset + 256] = x
    apart = torch.zeros(18, 9, device=DEV)
    apart[:, 2:8] = z
    oracle_out, bound = oracle.moe_layer(x, z.cpu(), up.cpu(), down.cpu(), 2, "swiglu")
    got = run(wide[:, offset:offset + 256], apart[:, 2:8], up, down, 2, "swiglu")
    oracle.assert_within(got, oracle_out, bound)
    oracle.assert_within(want, oracle_out, bound)
    oracle.assert_within(run(x.t().contiguous().t(), z.t().contiguous().t(), up, down, 2, "swiglu"), oracle_out, bound)


def island(t, lay, pad=0):
    """t at an odd address (2 bytes past a multiple of 4), rows pad elements apart, NaN all around."""
    src = t.transpose(-2, -1) if lay == "cols" else t
    *front, rows, columns = src.shape
    count = src.numel() // max(columns, 1) if src.numel() else 0
    flat = torch.full((count * (columns + pad) + 18,), float("nan"), dtype=t.dtype, device=DEV)
    strides = [columns + pad, 1]
    for n in reversed(src.shape[1:-1]):
        strides.insert(0, strides[0] * n)
    view = torch.as_strided(flat, src.shape, strides[-src.dim():], 9)
    view.copy_(src)
    return view.transpose(-2, -1) if lay == "cols" else view


@pytest.mark.parametrize("H,I", [(8, 8), (9, 11), (63, 65), (130, 71), (65, 64), (1031, 519), (500, 2050)])
@pytest.mark.parametrize("lay", ["rows", "cols"])
@pytest.mark.parametrize("T", [1, 5, 20, 40])
def test_matrices_at_odd_addresses_among_nan(H, I, lay, T):
    for kind in ("silu", "swiglu", "interleaved") if I % 64 == 0 else ("silu", "swiglu"):
        x, z, up, down = make(T, 5, H, I, kind, dtype=HF)
        check(island(x, "rows", 3), z, island(up, lay), island(down, lay, 5), 2, kind)


def test_experts_that_share_their_weights():
    x, z, up, down = make(9, 5, 128, 64)
    up, down = up[:1].expand(5, -1, -1), down[:1].expand(5, -1, -1)
    check(x, z, up, down, 2, "swiglu")


def test_empty():
    x, z, up, down = make(0, 4, 64, 32)
    assert run(x, z, up, down, 2, "swiglu").shape == (0, 64)
    x, z, up, down = make(3, 4, 64, 0)
    assert torch.equal(run(x, z, up, down, 2, "swiglu"), torch.zeros_like(x))


@pytest.mark.parametrize("T,E,k,H,I,kind,lay", [(1, 128, 8, 2048, 768, "swiglu", "rows"), (32, 128, 8, 2048, 768, "swiglu", "cols"),
                                                (8, 8, 2, 4096, 14336, "interleaved", "rows"), (64, 16, 4, 2048, 1536, "silu", "rows")])
def test_sizes_of_served_layers(T, E, k, H, I, kind, lay):
    gen = torch.Generator(device=DEV).manual_seed(T)
    x = torch.randn(T, H, device=DEV, dtype=BF, generator=gen)
    z = torch.randn(T, E, device=DEV, generator=gen)
    shape_up, shape_down = (E, H, I if kind == "silu" else 2 * I), (E, I, H)
    swap = (lambda s: (s[0], s[2], s[1])) if lay == "cols" else (lambda s: s)
    up = torch.randn(swap(shape_up), device=DEV, dtype=BF, generator=gen).mul_(H ** -0.5)
    down = torch.randn(swap(shape_down), device=DEV, dtype=BF, generator=gen).mul_(I ** -0.5)
    if lay == "cols":
        up, down = up.transpose(1, 2), down.transpose(1, 2)
    got = run(x, z, up, down, k, kind)
    keep = [0, T // 2, T - 1][:T]                      # the oracle on some tokens: rows do not depend on one another
    want, bound = oracle.moe_layer(x[keep], z[keep].cpu(), up, down, k, kind)
    oracle.assert_within(got[keep], want, bound)


def test_near_the_layer_of_many_launches():
    """moe_forward rounds the product, the activation and each expert's result as well: four roundings against one."""
    x, z, up, down = make(32, 16, 512, 256)
    few, many = run(x, z, up, down, 4, "swiglu").float(), moe.moe_forward(x, z, up, down, 4).float()
    assert (few - many).norm() <= 4 * 2.0 ** -8 * many.norm()


def test_on_another_stream_and_in_a_graph():
    x, z, up, down = make(12, 24, 512, 256)
    want = run(x, z, up, down, 4, "swiglu")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(x, z, up, down, 4, "swiglu")
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = run(x, z, up, down, 4, "swiglu")
    for seed in range(1, 4):
        x2, z2, _, _ = make(12, 24, 512, 256, seed=seed)
        x.copy_(x2)
        z.copy_(z2)
        want = run(x, z, up, down, 4, "swiglu")
        held.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held, want)


def test_compiled_op_agrees():
    x, z, up, down = make(4, 8, 128, 64)
    assert torch.equal(torch.ops.grouped_mm_bf16_amd.few(x, z, up, down, 2, 1, True), run(x, z, up, down, 2, "swiglu"))
    torch.library.opcheck(torch.ops.grouped_mm_bf16_amd.few, (x, z, up, down, 2, 1, True), test_utils=("test_schema", "test_faketensor"))
