"""Products of 8-bit integers on a real MI355X against exact sums: sizes around the tiles and steps, odd ones, strides and alignments, groups of any
length, gathered rows, all types; the rounding of rows bit for bit; the expert layer; captured, on another stream, compiled."""
import pytest
import torch

from grouped_mm_bf16_amd import int8, kernels
from oracle import int8_oracle as oracle
from oracle import operators_oracle as plain

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF, SF = torch.bfloat16, torch.float16, torch.float32


def values(gen, *shape, low=-128):
    return torch.randint(low, 128, shape, generator=gen, dtype=torch.int8).to(DEV)


def scales(gen, *shape):
    return (0.5 + torch.rand(*shape, generator=gen)).to(DEV) * 1e-2


def make(M, K, N, groups=None, seed=0, pad=0, low=-128):
    """pad: bytes that rows and columns lie further apart, odd numbers among them; what lies between is no zero."""
    gen = torch.Generator().manual_seed(seed + 7 * M + 3 * K + N)
    a = int8.Rows(values(gen, M, K + pad, low=low)[:, :K], scales(gen, M))
    lead = () if groups is None else (groups,)
    b = int8.Columns(values(gen, *lead, N, K + pad, low=low)[..., :K].transpose(-2, -1), scales(gen, *lead, N))
    return a, b


def check(a, b, dtype=BF):
    out = int8.int8_mm(a, b, dtype)
    assert out.dtype == dtype and out.is_contiguous()
    want, bound = oracle.mm(a.values, a.scale, b.values, b.scale, dtype)
    plain.assert_within(out, want, bound)
    return out


# ------------------------------------------------------------------ rounding
def check_rounding(x):
    got = int8.quantize_rows(x)
    q, scale = oracle.quantize(x)
    assert got.values.shape == x.shape and got.values.stride(0) % 16 == 0
    finite = torch.isfinite(scale)
    assert torch.equal(got.scale.cpu()[finite], scale[finite]) and torch.equal(got.scale.cpu().isnan(), scale.isnan())
    assert torch.equal(got.scale.cpu().isinf(), scale.isinf())
    assert torch.equal(got.values.cpu().double(), q)
    return got


@pytest.mark.parametrize("width", [1, 3, 15, 16, 17, 255, 256, 257, 1000, 1024, 1031, 2048, 2056, 4096, 4100, 8192, 8209, 16384, 16400, 40001])
@pytest.mark.parametrize("dtype", [BF, HF, SF])
def test_rounding(width, dtype):
    gen = torch.Generator().manual_seed(width)
    check_rounding((torch.randn(9, width, generator=gen) * torch.logspace(-3, 3, 9)[:, None]).to(dtype).to(DEV))


@pytest.mark.parametrize("rows", [1, 2, 5, 300, 70000])
def test_rounding_of_rows(rows):
    gen = torch.Generator().manual_seed(rows)
    check_rounding(torch.randn(rows, 72, generator=gen).to(BF).to(DEV))


def test_rounding_of_ties_zeros_and_extremes():
    """Halves of a step go to the even neighbour; rows of zeros, subnormal ones, the largest values."""
    half = torch.arange(-254, 255).float() / 2
    rows = [half, half * 2.0 ** -90, half * 2.0 ** -96, half * 2.0 ** -140, torch.zeros(509), half / 127 * 3.3e38, torch.full((509,), -1e-30), half * 2.0 ** 100]
    check_rounding(torch.stack(rows).to(DEV))
    check_rounding(half[None].to(BF).to(DEV))


def test_rounding_of_what_is_no_number():
    x = torch.randn(5, 300)
    x[1, 7], x[2, 299], x[3, 0] = float("inf"), float("nan"), -float("inf")
    x[3, 5] = float("nan")
    got = check_rounding(x.to(DEV))
    b = int8.quantize_columns(torch.randn(300, 64, device=DEV))
    out = int8.int8_mm(got, b, SF)
    assert torch.equal(out.isnan().all(1).cpu(), torch.tensor([False, True, True, True, False])) and torch.isfinite(out[[0, 4]]).all()


@pytest.mark.parametrize("pad,offset", [(1, 0), (3, 1), (8, 0)])
@pytest.mark.parametrize("dtype", [BF, SF])
def test_rounding_of_rows_that_lie_apart(pad, offset, dtype):
    wide = torch.randn(20, 130 + pad + offset, device=DEV).to(dtype)
    check_rounding(wide[:, offset:130 + offset])
    check_rounding(torch.randn(130, 20, device=DEV).to(dtype).t())


@pytest.mark.parametrize("shape", [(40, 24), (3, 40, 24), (2, 33, 17), (0, 8, 8), (5, 0), (3, 0, 4), (4, 4, 0)])
@pytest.mark.parametrize("turned", [False, True])
def test_rounding_of_columns(shape, turned):
    w = torch.randn(*shape, device=DEV, dtype=BF)
    if turned:
        w = torch.randn(*shape[:-2], shape[-1], shape[-2], device=DEV, dtype=BF).transpose(-2, -1)
    got = int8.quantize_columns(w)
    assert got.values.shape == shape and got.scale.shape == shape[:-2] + shape[-1:]
    q, scale = oracle.quantize(w.transpose(-2, -1).reshape(-1, shape[-2]) if w.numel() else torch.zeros(got.scale.numel(), shape[-2]))
    assert torch.equal(got.values.transpose(-2, -1).reshape(-1, shape[-2]).cpu().double() if w.numel() else q, q) and torch.equal(got.scale.reshape(-1).cpu(), scale)


# ------------------------------------------------------------------ one matrix
@pytest.mark.parametrize("K", [1, 2, 15, 16, 17, 31, 63, 64, 65, 127, 128, 129, 143, 255, 384, 1000, 1031, 4096])
@pytest.mark.parametrize("M", [1, 20, 70, 300])
def test_depths(M, K):
    check(*make(M, K, 136))


@pytest.mark.parametrize("N", [1, 2, 7, 8, 9, 15, 16, 33, 64, 127, 129, 255, 256, 257, 260, 519, 1000])
@pytest.mark.parametrize("dtype", [BF, HF, SF])
def test_columns(N, dtype):
    for M in (5, 90):
        check(*make(M, 200, N), dtype)


@pytest.mark.parametrize("M", [1, 2, 15, 16, 17, 31, 33, 48, 63, 64, 65, 127, 128, 129, 200, 256, 257, 700, 1025])
@pytest.mark.parametrize("N", [64, 520])
def test_rows(M, N):
    check(*make(M, 320, N))


@pytest.mark.parametrize("dtype", [BF, HF, SF])
@pytest.mark.parametrize("M,K,N", [(513, 777, 1301), (2100, 512, 2304), (64, 8192, 640), (48, 8191, 200)])
def test_sizes(M, K, N, dtype):
    check(*make(M, K, N), dtype)


@pytest.mark.parametrize("pad", [1, 8, 16, 40])
@pytest.mark.parametrize("M", [3, 80])
@pytest.mark.parametrize("K", [64, 100, 101])
def test_rows_and_columns_that_lie_apart(M, K, pad):
    check(*make(M, K, 72, pad=pad))


def test_operands_at_any_address():
    gen = torch.Generator().manual_seed(0)
    for offset in (1, 4, 16):
        a = int8.Rows(values(gen, 50 * 96 + 64)[offset:offset + 50 * 96].view(50, 96), scales(gen, 51)[1:])
        b = int8.Columns(values(gen, 40 * 96 + 64)[offset:offset + 40 * 96].view(40, 96).t(), scales(gen, 41)[1:])
        check(a, b)


def test_the_largest_sums():
    """-128 times -128 as often as K allows, and its neighbour of the other sign."""
    K = int8.MAX_K
    for M in (2, 70):
        a = int8.Rows(torch.full((M, K), -128, dtype=torch.int8, device=DEV), torch.ones(M, device=DEV))
        b = int8.Columns(torch.full((3, K), -128, dtype=torch.int8, device=DEV).t(), torch.ones(3, device=DEV))
        b.values[:, 1] = 127
        check(a, b, SF)


@pytest.mark.parametrize("M,K,N", [(0, 64, 64), (5, 64, 0), (5, 0, 8), (100, 0, 300)])
def test_nothing(M, K, N):
    a, b = make(M, K, N)
    out = int8.int8_mm(a, b)
    assert out.shape == (M, N) and not out.any()


def test_scales_of_any_size():
    a, b = make(70, 128, 64)
    a.scale[0], a.scale[1], a.scale[2] = 0.0, float("inf"), 1e38
    b.scale[3] = float("nan")
    out = int8.int8_mm(a, b, SF)
    want, _ = oracle.mm(a.values, a.scale, b.values, b.scale, SF)
    want = want.float()      # beyond fp32's range: infinite
    assert torch.equal(out.isnan().cpu(), want.isnan()) and torch.equal(out.isinf().cpu(), want.isinf())


# ------------------------------------------------------------------ groups
def check_groups(sizes, K, N, dtype=BF, extra=0, gather=None, seed=0, pad=0):
    M = sum(sizes) + extra
    a, b = make(gather or M, K, N, len(sizes), seed, pad)
    offs = torch.tensor(sizes).cumsum(0).to(torch.int32).to(DEV)
    index = None
    if gather:
        index = torch.randint(-1, gather + 1, (M,), generator=torch.Generator().manual_seed(seed)).to(torch.int32).to(DEV)
    out = int8.grouped_int8_mm(a, b, offs, dtype, index)
    want, bound, owned = oracle.grouped_mm(a.values, a.scale, b.values, b.scale, offs, dtype, index)
    plain.assert_within(out[owned.to(DEV)], want[owned], bound[owned])
    return out


GROUPS = [[5], [0, 7, 0, 1, 30, 0], [64, 65, 1, 128, 129], [300, 0, 0, 513, 2], [1] * 40, [3, 0] * 20, [0, 0, 0], [17, 200, 5, 90, 256, 31]]


@pytest.mark.parametrize("sizes", GROUPS)
@pytest.mark.parametrize("dtype", [BF, HF, SF])
def test_groups(sizes, dtype):
    check_groups(sizes, 192, 264, dtype)
    check_groups(sizes, 77, 100, dtype, extra=9)


@pytest.mark.parametrize("sizes", GROUPS)
@pytest.mark.parametrize("source", [1, 50, 400])
def test_gathered_rows(sizes, source):
    check_groups(sizes, 160, 136, gather=source)
    check_groups(sizes, 97, 136, gather=source, pad=15)


def test_very_many_groups():
    sizes = [(g * 7) % 5 for g in range(1023)]
    check_groups(sizes, 64, 40)
    check_groups(sizes, 64, 40, gather=100)


def test_malformed_offsets():
    """Group g is offs[g - 1] .. offs[g] - 1, clamped to the rows there are: nothing outside is read or written, and a row that one group alone claims is
    that group's (one that two claim is either's)."""
    a, b = make(100, 64, 64, 3)
    for offs in ([10, 20, 30], [50, 20, 60], [-5, 40, 300], [100, 100, 100], [300, -7, 50]):
        out = int8.grouped_int8_mm(a, b, torch.tensor(offs, dtype=torch.int32, device=DEV))
        ends = [0] + [min(max(end, 0), 100) for end in offs]
        claims = torch.zeros(100, dtype=torch.int32)
        for first, end in zip(ends, ends[1:]):
            claims[first:max(first, end)] += 1
        for g, (first, end) in enumerate(zip(ends, ends[1:])):
            if end > first:
                want, bound = oracle.mm(a.values[first:end], a.scale[first:end], b.values[g], b.scale[g], BF)
                alone = claims[first:end] == 1
                plain.assert_within(out[first:end][alone.to(DEV)], want[alone], bound[alone])


def test_one_matrix_for_all_groups():
    a, b = make(90, 128, 64, 1)
    wide = int8.Columns(b.values.expand(4, -1, -1), b.scale.expand(4, -1).contiguous())
    offs = torch.tensor([20, 20, 70, 90], dtype=torch.int32, device=DEV)
    assert torch.equal(int8.grouped_int8_mm(a, wide, offs), int8.int8_mm(a, int8.Columns(b.values[0], b.scale[0])))


@pytest.mark.parametrize("M,K,N", [(300, 8192, 512), (1100, 8190, 2300), (130, 16384, 4096)])
def test_tiles_cut_along_k(M, K, N):
    """With a workspace the last round's tiles are cut: exact sums, so not a bit changes."""
    a, b = make(M, K, N)
    for dtype in (BF, HF, SF):
        with kernels.tail_split(True):
            cut = check(a, b, dtype)
        with kernels.tail_split(False):
            assert torch.equal(int8.int8_mm(a, b, dtype), cut)
    sizes = [M // 3, 0, M - M // 3]
    check_groups(sizes, K, N, gather=M)


# ------------------------------------------------------------------ linear layer, expert layer
@pytest.mark.parametrize("dtype", [BF, HF, SF])
@pytest.mark.parametrize("T", [1, 4, 16, 33, 64, 65, 300])
def test_linear(T, dtype):
    gen = torch.Generator().manual_seed(T)
    x, w = torch.randn(T, 328, generator=gen).to(dtype).to(DEV), torch.randn(200, 328, generator=gen).to(dtype).to(DEV).t()
    columns = int8.quantize_columns(w)
    out = int8.linear_int8(x, columns)
    q, scale = oracle.quantize(x)
    plain.assert_within(out, *oracle.mm(q, scale, columns.values, columns.scale, dtype))
    assert torch.equal(out, int8.int8_mm(int8.quantize_rows(x), columns, dtype))
    # what the roundings to 8 bits leave: half a step of either operand, as if at random, against values of a deviation of one
    full = x.double() @ w.double()
    assert (out.double() - full).norm() <= 0.03 * full.norm()


def layer(T, E, H, inner, kind, dtype=BF, seed=0):
    gen = torch.Generator().manual_seed(seed + T)
    x, z = torch.randn(T, H, generator=gen).to(dtype).to(DEV), torch.randn(T, E, generator=gen).to(DEV)
    up = int8.quantize_columns((torch.randn(E, inner * (2 if kind == "swiglu" else 1), H, generator=gen) * H ** -0.5).to(dtype).to(DEV).transpose(1, 2))
    down = int8.quantize_columns((torch.randn(E, H, inner, generator=gen) * inner ** -0.5).to(dtype).to(DEV).transpose(1, 2))
    return x, z, up, down


@pytest.mark.parametrize("kind", ["silu", "swiglu"])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("T,E,k,H,inner", [(1, 4, 2, 64, 64), (7, 128, 8, 256, 128), (33, 6, 2, 130, 70), (64, 8, 2, 512, 768), (200, 12, 3, 136, 72), (700, 16, 4, 256, 128)])
def test_layer(T, E, k, H, inner, dtype, kind):
    """The experts' rows and their sum are rounded to x's type.  The activations' last bits of fp32 decide a value's step of 8 bits where it lies within
    2^-18 of a half: one in a thousand values at most is a step (an eighth of their deviation at most) off, that is 2^-8 of the result."""
    x, z, up, down = layer(T, E, H, inner, kind, dtype)
    out = int8.moe_forward_int8(x, z, up, down, k, kind)
    want = oracle.layer(x, z, up.values, up.scale, down.values, down.scale, k, kind)
    assert out.dtype == dtype and out.shape == x.shape
    assert (plain.f64(out) - want).norm() <= (2.5 * plain.UNIT[dtype] + 2.0 ** -8) * want.norm()


@pytest.mark.parametrize("T,E,k,H,inner", [(65, 4, 2, 64, 64), (129, 3, 3, 333, 192), (400, 8, 2, 320, 192), (900, 5, 2, 1031, 320), (2500, 128, 8, 192, 64),
                                           (1500, 4, 2, 512, 1024)])
def test_layer_whose_first_product_activates(T, E, k, H, inner):
    """Inner sizes of whole blocks of 64: SwiGLU in the tile's epilogue, tiles of every height."""
    x, z, up, down = layer(T, E, H, inner, "swiglu")
    out = int8.moe_forward_int8(x, z, up, down, k)
    want = oracle.layer(x, z, up.values, up.scale, down.values, down.scale, k, "swiglu")
    assert (plain.f64(out) - want).norm() <= (2.5 * 2.0 ** -8 + 2.0 ** -8) * want.norm()
    # the two products of the layer one after the other, the first without the epilogue: the same but for the activation's last bits
    r = int8.moe.moe_route(z, k)
    a = int8.quantize_rows(x)
    h = int8.grouped_int8_mm(a, up, r.offs, SF, r.row_token)
    fused = int8._activated(a, r, up.values, up.scale, 1)
    apart = int8._gated_now(h, 1)
    # e^-g to a few units of fp32 of its exponent, |g| below 30; the maximum of the row alone stands in the scale
    assert ((fused[1] - apart[1]).abs() <= 2.0 ** -18 * apart[1]).all()
    step = (fused[0][:, :inner].int() - apart[0][:, :inner].int()).abs()
    assert step.max() <= 1 and step.float().mean() <= 1e-3


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("T,E,k,H,inner", [(1, 128, 8, 2048, 768), (2, 40, 8, 130, 64), (16, 4, 1, 72, 128), (5, 3, 3, 2056, 200), (8, 2, 2, 1034, 66), (1, 16, 16, 16, 16),
                                           (1, 1, 1, 4096, 32), (17, 6, 1, 136, 64)])
def test_layer_of_a_few_slots(T, E, k, H, inner, dtype):
    """The second product's last workgroups add up the result: strips that end inside, experts without rows, on one workspace again and again."""
    for seed in range(3):
        x, z, up, down = layer(T, E, H, inner, "swiglu", dtype, seed)
        out = int8.moe_forward_int8(x, z, up, down, k)
        want = oracle.layer(x, z, up.values, up.scale, down.values, down.scale, k, "swiglu")
        assert (plain.f64(out) - want).norm() <= (2.5 * plain.UNIT[dtype] + 2.0 ** -8) * want.norm()
        for _ in range(5):
            assert torch.equal(int8.moe_forward_int8(x, z, up, down, k), out)


@pytest.mark.parametrize("dtype", [BF, HF, SF])
@pytest.mark.parametrize("M", [65, 80, 96, 97, 128, 129, 192, 193, 250, 256, 257])
@pytest.mark.parametrize("K,N", [(136, 200), (1024, 64), (2050, 72), (4096, 1000), (16384, 136)])
def test_blocks_of_rows(M, K, N, dtype):
    """One matrix streamed past several blocks of rows, the last one shorter; long columns in parts; sums are exact, whatever computes them."""
    a, b = make(M, K, N)
    out = check(a, b, dtype)
    for rows in (slice(0, 64), slice(64, 65), slice(M - 3, M)):
        assert torch.equal(out[rows], int8.int8_mm(int8.Rows(a.values[rows], a.scale[rows]), b, dtype))


@pytest.mark.parametrize("M,G,largest", [(65, 3, 60), (100, 40, 7), (128, 4, 128), (300, 10, 33), (512, 128, 100), (1000, 50, 49), (1024, 32, 48), (1024, 1023, 65), (1025, 64, 20),
                                          (700, 21, 700)])
def test_blocks_of_rows_of_groups(M, G, largest):
    """Groups of none, one, exactly a block, a block and one, many blocks; either side of the limits."""
    gen = torch.Generator().manual_seed(M + G)
    sizes = torch.bincount(torch.randint(0, G, (M - largest,), generator=gen), minlength=G)
    sizes[G // 2] += largest
    check_groups(sizes.tolist(), 130, 72)
    check_groups(sizes.tolist(), 1024, 264, gather=M)


@pytest.mark.parametrize("kind", ["silu", "swiglu"])
@pytest.mark.parametrize("T,E,k,H,inner", [(17, 3, 3, 136, 64), (33, 40, 8, 256, 128), (64, 8, 8, 130, 70), (64, 5, 2, 512, 256), (65, 8, 2, 256, 128), (96, 8, 2, 1040, 72),
                                           (128, 8, 2, 256, 192), (130, 8, 2, 64, 64), (200, 128, 8, 128, 64), (255, 64, 8, 72, 128), (256, 64, 8, 136, 64), (256, 300, 32, 64, 32),
                                           (257, 64, 8, 64, 64)])
def test_layer_of_blocks_of_rows(T, E, k, H, inner, kind):
    """Experts of more rows than a block, of a few and of none; either side of every limit.  A skewed choice gives one expert all tokens."""
    x, z, up, down = layer(T, E, H, inner, kind)
    for skew in (False, True):
        if skew:
            z = z.clone()
            z[:, E // 2] += 20
        out = int8.moe_forward_int8(x, z, up, down, k, kind)
        want = oracle.layer(x, z, up.values, up.scale, down.values, down.scale, k, kind)
        assert (plain.f64(out) - want).norm() <= (2.5 * 2.0 ** -8 + 2.0 ** -8) * want.norm()
        assert torch.equal(int8.moe_forward_int8(x, z, up, down, k, kind), out)


def test_layer_over_all_experts_and_halves_of_logits():
    x, z, up, down = layer(40, 10, 64, 64, "swiglu")
    out = int8.moe_forward_int8(x, z.to(BF), up, down, 3, renormalize=False)
    want = oracle.layer(x, z.to(BF), up.values, up.scale, down.values, down.scale, 3, "swiglu", False)
    assert (plain.f64(out) - want).norm() <= 2.0 ** -6 * want.norm()


@pytest.mark.parametrize("T", [1, 6, 90])
def test_layer_of_operands_that_lie_elsewhere(T):
    """Rows apart, transposed ones, logits of which neither is contiguous, weights of experts far apart and at odd addresses."""
    x, z, up, down = layer(T, 6, 136, 64, "swiglu")
    want = int8.moe_forward_int8(x, z, up, down, 2)
    apart = torch.zeros(T, 150, dtype=BF, device=DEV)[:, 3:139].copy_(x)
    turned = x.t().contiguous().t()
    far = lambda c: int8.Columns(torch.zeros(6, 3, *c.values.transpose(1, 2).shape[1:], dtype=torch.int8, device=DEV)[:, 1].copy_(c.values.transpose(1, 2)).transpose(1, 2), c.scale)
    odd = lambda c: int8.Columns(torch.zeros(c.values.numel() + 1, dtype=torch.int8, device=DEV)[1:].reshape(c.values.transpose(1, 2).shape)
                                 .copy_(c.values.transpose(1, 2)).transpose(1, 2), c.scale)
    for rows in (apart, turned):
        for logits in (z.t().contiguous().t(), torch.zeros(T, 9, device=DEV)[:, 2:8].copy_(z)):
            for place in (far, odd):
                assert torch.equal(int8.moe_forward_int8(rows, logits, place(up), place(down), 2), want)


def test_layer_of_nothing():
    x, z, up, down = layer(3, 4, 64, 64, "swiglu")
    assert int8.moe_forward_int8(x[:0], z[:0], up, down, 2).shape == (0, 64)


@pytest.mark.parametrize("T", [4, 100, 600])
def test_captured_and_replayed(T):
    x, z, up, down = layer(T, 8, 256, 128, "swiglu")
    columns = int8.Columns(up.values[0], up.scale[0])
    run = lambda: (int8.moe_forward_int8(x, z, up, down, 2), int8.linear_int8(x, columns))
    run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = run()
    for seed in range(1, 4):
        x2, z2, _, _ = layer(T, 8, 256, 128, "swiglu", seed=seed)
        x.copy_(x2)
        z.copy_(z2)
        want = run()
        for t in held:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(held, want))


@pytest.mark.parametrize("M", [40, 100, 256])
def test_captured_where_few_rows_are_cut(M):
    """Parts of k lie in a workspace: the graphs' own, so they do not meet each other's or the eager calls'."""
    a, b = make(M, 16384, 136)
    other = int8.Rows(a.values.flip(0).contiguous(), a.scale)
    want, want_other = int8.int8_mm(a, b), int8.int8_mm(other, b)
    graphs = []
    for rows in (a, other):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = int8.int8_mm(rows, b)
        graphs.append((graph, held))
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(4):
        for _, held in graphs:
            held.zero_()
        torch.cuda.synchronize()
        for (graph, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        eager = int8.int8_mm(a, b)
        torch.cuda.synchronize()
        assert torch.equal(eager, want) and torch.equal(graphs[0][1], want) and torch.equal(graphs[1][1], want_other)


def test_captured_where_tiles_are_cut():
    a, b = make(300, 8192, 512)
    int8.int8_mm(a, b)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = int8.int8_mm(a, b)
        graphs.append((graph, held))
    want = int8.int8_mm(a, b)
    for _ in range(3):
        for graph, held in graphs:
            held.zero_()
        for graph, _ in graphs:
            graph.replay()
        assert torch.equal(int8.int8_mm(a, b), want)
        torch.cuda.synchronize()
        assert all(torch.equal(held, want) for _, held in graphs)


def test_on_two_streams_at_once():
    a, b = make(300, 8192, 512)
    x, z, up, down = layer(30, 8, 256, 128, "swiglu")
    want = int8.int8_mm(a, b), int8.moe_forward_int8(x, z, up, down, 2)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                got.append((int8.int8_mm(a, b), int8.moe_forward_int8(x, z, up, down, 2)))
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for g in got for p, q in zip(g, want))


@pytest.mark.parametrize("T", [5, 90])
def test_compiled(T):
    x, z, up, down = layer(T, 8, 128, 64, "swiglu")

    def f(x_, z_, uv, us, dv, ds):
        y = int8.moe_forward_int8(x_ * 2, z_, int8.Columns(uv, us), int8.Columns(dv, ds), 2)
        return y + int8.linear_int8(x_, int8.Columns(uv[0], us[0])) + 1, int8.int8_mm(int8.quantize_rows(x_), int8.Columns(uv[1], us[1]), torch.float32)

    torch._dynamo.reset()
    args = (x, z, *up, *down)
    for p, q in zip(f(*args), torch.compile(f, backend="aot_eager", fullgraph=True)(*args)):
        assert torch.equal(p, q)
