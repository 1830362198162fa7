"""The projection with many requests' adapters on a real MI355X, forward and backward, against the formulas in 64 bits: numbers of rows
around the kernels' sixteens, sizes without alignment, ranks, layouts, which rows have which adapter; gradients also against
differences."""
import pytest
import torch

from grouped_mm_bf16_amd import lora
from oracle import operators_oracle as oracle

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF = torch.bfloat16, torch.float16


def matrix(gen, shape, dtype, scale, lay):
    """lay: rows, cols (last two dimensions swapped in memory), any (no dimension contiguous)."""
    if lay == "cols":
        return matrix(gen, (*shape[:-2], shape[-1], shape[-2]), dtype, scale, "rows").transpose(-2, -1)
    if lay == "any":
        return (torch.randn(*shape[:-1], 2 * shape[-1] + 1, generator=gen) * scale).to(dtype).to(DEV)[..., 1::2]
    return (torch.randn(*shape, generator=gen) * scale).to(dtype).to(DEV)


def make(T, K, N, R, L, lay="rows", lay_w=None, dtype=BF, pattern="mixed", seed=0, pad=0, offset=0):
    gen = torch.Generator().manual_seed(seed + T + K + N + R + L)
    x = torch.randn(T, K + pad + offset, generator=gen).to(dtype).to(DEV)[:, offset:offset + K]
    weight = matrix(gen, (K, N), dtype, max(K, 1) ** -0.5, lay_w or ("rows" if lay == "any" else lay))
    a, b = matrix(gen, (L, K, R), dtype, max(K, 1) ** -0.5, lay), matrix(gen, (L, R, N), dtype, R ** -0.5, lay)
    if pattern == "mixed":
        adapter = torch.randint(-1, L, (T,), generator=gen)
    elif pattern == "requests":
        adapter = (torch.arange(T) * (L + 1) // max(T, 1)) - 1
    elif pattern == "one":
        adapter = torch.full((T,), L - 1)
    else:
        adapter = torch.full((T,), -1)
    scale = 0.5 + torch.rand(L, generator=gen)
    return x, weight, a, b, adapter.to(torch.int32).to(DEV), scale.to(DEV)


def check(x, weight, a, b, adapter, scale):
    got = lora.lora_linear(x, weight, a, b, adapter, scale)
    assert got.dtype == x.dtype and got.shape == (x.size(0), weight.size(1))
    want, bound = oracle.lora_linear(x, weight, a, b, adapter, scale)
    oracle.assert_within(got, want, bound, "out")
    assert torch.equal(got, lora.lora_linear(x, weight, a, b, adapter, scale)), "not the same twice"
    return got


def check_grads(x, weight, a, b, adapter, scale, seed=1, need=(True, False, True, True)):
    gen = torch.Generator().manual_seed(seed)
    dy = torch.randn(x.size(0), weight.size(1), generator=gen).to(x.dtype).to(DEV)
    leaves = [t.detach().requires_grad_(n) for t, n in zip((x, weight, a, b), need)]
    y = lora.lora_linear(*leaves, adapter, scale)
    oracle.assert_within(y, *oracle.lora_linear(x, weight, a, b, adapter, scale), "out")
    grads = iter(torch.autograd.grad(y, [t for t, n in zip(leaves, need) if n], dy))
    for name, leaf, n, (want, bound) in zip(("dx", "dweight", "da", "db"), leaves, need,
                                            oracle.lora_backward(dy, x, weight, a, b, adapter, scale)):
        if n:
            got = next(grads)
            assert got.shape == leaf.shape and got.dtype == leaf.dtype
            oracle.assert_within(got, want, bound, name)


ROWS = [1, 2, 15, 16, 17, 32, 33, 48, 63, 64, 65, 80, 200, 256, 257, 272, 515]


@pytest.mark.parametrize("T", ROWS)
@pytest.mark.parametrize("pattern", ["mixed", "requests"])
def test_numbers_of_rows(T, pattern):
    check(*make(T, 512, 384, 16, 9, pattern=pattern))


@pytest.mark.parametrize("T", [3, 40, 130, 300])
@pytest.mark.parametrize("lay", ["rows", "cols", "any"])
@pytest.mark.parametrize("lay_w", ["rows", "cols"])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_layouts(T, lay, lay_w, dtype):
    check(*make(T, 320, 264, 24, 4, lay, lay_w, dtype))


@pytest.mark.parametrize("R", [1, 2, 4, 5, 8, 16, 31, 32, 40, 64, 100, 128, 129, 200, 256])
@pytest.mark.parametrize("T,lay", [(20, "rows"), (20, "cols"), (330, "rows"), (330, "cols")])
def test_ranks(R, T, lay):
    check(*make(T, 256, 192, R, 5, lay))


@pytest.mark.parametrize("K,N", [(1, 1), (8, 8), (7, 5), (64, 130), (130, 64), (255, 33), (1031, 519), (2048, 136), (136, 2056), (4096, 4096)])
@pytest.mark.parametrize("T,lay", [(5, "rows"), (5, "cols"), (90, "rows"), (290, "cols")])
def test_sizes(K, N, T, lay):
    check(*make(T, K, N, 12, 3, lay))


@pytest.mark.parametrize("T", [10, 100, 400])
@pytest.mark.parametrize("pad,offset", [(8, 0), (3, 0), (0, 1)])
def test_rows_of_x_that_lie_apart(T, pad, offset):
    check(*make(T, 256, 128, 16, 4, pad=pad, offset=offset))


def island(t, lay, pad=0):
    """t at an odd address (2 bytes past a multiple of 4), rows pad elements apart, NaN all around."""
    src = t.transpose(-2, -1) if lay == "cols" else t
    rows, columns = src.shape[:-1].numel(), src.size(-1)
    flat = torch.full((rows * (columns + pad) + 18,), float("nan"), dtype=t.dtype, device=DEV)
    strides = [columns + pad, 1] if src.dim() == 2 else [src.size(1) * (columns + pad), columns + pad, 1]
    view = torch.as_strided(flat, src.shape, strides, 9)
    view.copy_(src)
    return view.transpose(-2, -1) if lay == "cols" else view


@pytest.mark.parametrize("K,N,R", [(8, 8, 8), (9, 11, 9), (65, 130, 31), (254, 261, 33), (1031, 519, 12), (3000, 77, 100)])
@pytest.mark.parametrize("T", [1, 20, 40, 130, 300])
@pytest.mark.parametrize("lay", ["rows", "cols"])
def test_matrices_at_odd_addresses_among_nan(K, N, R, T, lay):
    x, weight, a, b, adapter, scale = make(T, K, N, R, 3, dtype=HF)
    x, weight, a, b = island(x, "rows", 3), island(weight, lay), island(a, lay, 5), island(b, lay)
    check(x, weight, a, b, adapter, scale)
    if T in (40, 300):
        check_grads(x, weight, a, b, adapter, scale)


@pytest.mark.parametrize("T", [6, 100, 400])
@pytest.mark.parametrize("pattern", ["one", "none"])
def test_one_adapter_or_none(T, pattern):
    x, weight, a, b, adapter, scale = make(T, 256, 128, 16, 4, pattern=pattern)
    got = check(x, weight, a, b, adapter, scale)
    check(x, weight, a, b, adapter, None)
    if pattern == "none":      # neither adapters nor scales are looked at
        a, b, scale = (t.fill_(float("nan")) for t in (a, b, scale))
        assert torch.equal(lora.lora_linear(x, weight, a, b, adapter, scale), got)
        check(x, weight, a[:0], b[:0], torch.zeros_like(adapter), scale[:0])


@pytest.mark.parametrize("T", [6, 100, 400])
def test_numbers_outside_the_adapters_mean_none(T):
    x, weight, a, b, adapter, scale = make(T, 128, 64, 8, 4)
    want = lora.lora_linear(x, weight, a, b, adapter, scale)
    for far in (4, 1 << 30, -5, -(1 << 31)):
        assert torch.equal(lora.lora_linear(x, weight, a, b, torch.where(adapter < 0, far, adapter).to(torch.int32), scale), want)


@pytest.mark.parametrize("T", [6, 100, 400])
def test_adapters_that_are_not_finite_stay_with_their_rows(T):
    x, weight, a, b, adapter, scale = make(T, 128, 64, 8, 4)
    adapter[0], adapter[1] = 2, 1
    want = lora.lora_linear(x, weight, a, b, adapter, scale)
    a[2, 0, 0], b[2, 1, 5] = float("nan"), float("inf")
    got = lora.lora_linear(x, weight, a, b, adapter, scale)
    others = adapter != 2
    assert torch.equal(got[others], want[others]) and not torch.isfinite(got[~others]).all()


def test_many_adapters():
    check(*make(60, 64, 64, 8, 1022))
    check_grads(*make(600, 64, 64, 8, 1022))


# ------------------------------------------------------------------ gradients
@pytest.mark.parametrize("T", [1, 2, 16, 40, 64, 65, 129, 300, 513, 1025])
@pytest.mark.parametrize("pattern", ["mixed", "requests", "one"])
def test_gradients(T, pattern):
    check_grads(*make(T, 256, 192, 16, 5, pattern=pattern))


@pytest.mark.parametrize("R", [1, 5, 8, 17, 32, 64, 65, 128, 256])
def test_gradients_of_ranks(R):
    check_grads(*make(150, 136, 264, R, 3))


@pytest.mark.parametrize("K,N", [(8, 8), (7, 5), (130, 64), (1031, 519), (2056, 136), (1, 300)])
@pytest.mark.parametrize("lay", ["rows", "cols", "any"])
def test_gradients_of_sizes_and_layouts(K, N, lay):
    check_grads(*make(100, K, N, 12, 3, lay, "rows", HF))


def test_gradients_of_adapters_with_few_rows_many_rows_and_none():
    """One adapter has rows for several chunks, one exactly one chunk, some a few, one none; all rows in random order."""
    x, weight, a, b, adapter, scale = make(2300, 72, 136, 16, 8)
    adapter = torch.cat([torch.full((n,), i) for i, n in ((0, 1200), (1, 512), (2, 513), (3, 1), (5, 9), (6, 57), (-1, 8))])
    order = torch.randperm(2300, generator=torch.Generator().manual_seed(0))
    adapter = adapter[order].to(torch.int32).to(DEV)
    check_grads(x, weight, a, b, adapter, scale)
    leaf = b.detach().requires_grad_()
    grad, = torch.autograd.grad(lora.lora_linear(x, weight, a, leaf, adapter, scale), leaf, torch.ones(2300, 136, dtype=BF, device=DEV))
    assert torch.equal(grad[[4, 7]], torch.zeros_like(grad[[4, 7]]))


@pytest.mark.parametrize("need", [(True, False, False, False), (False, False, True, False), (False, False, False, True),
                                  (False, True, False, False), (True, True, True, True), (False, False, True, True)])
@pytest.mark.parametrize("T", [20, 100])
def test_some_gradients_only(need, T):
    check_grads(*make(T, 128, 96, 8, 3), need=need)


def test_gradients_have_their_parameters_layout_and_are_the_same_every_time():
    x, weight, a, b, adapter, scale = make(700, 128, 192, 16, 4, "cols")
    dy = torch.randn(700, 192, generator=torch.Generator().manual_seed(3)).to(BF).to(DEV)
    leaves = [t.detach().requires_grad_() for t in (x, a, b)]
    once, again = (torch.autograd.grad(lora.lora_linear(leaves[0], weight, *leaves[1:], adapter, scale), leaves, dy) for _ in range(2))
    assert once[1].stride() == a.stride() and once[2].stride() == b.stride()
    assert all(torch.equal(p, q) for p, q in zip(once, again))


def test_gradients_when_other_rows_are_not_finite():
    """Rows of one adapter do not reach the gradients of another."""
    x, weight, a, b, adapter, scale = make(90, 64, 64, 8, 3)
    dy = torch.randn(90, 64, generator=torch.Generator().manual_seed(3)).to(BF).to(DEV)
    grads = []
    for bad in (False, True):
        if bad:
            x[adapter == 1], dy[adapter == 1] = float("nan"), float("inf")
            x[adapter == -1] = float("nan")
        leaves = [t.detach().requires_grad_() for t in (a, b)]
        grads.append(torch.autograd.grad(lora.lora_linear(x, weight, *leaves, adapter, scale), leaves, dy))
    for p, q in zip(*grads):
        assert torch.equal(p[[0, 2]], q[[0, 2]]) and not torch.isfinite(q[1]).any()


def test_gradients_against_differences():
    """Central differences of the formula in 64 bits (it is a product of three factors: exact up to rounding); the gradients are in
    fp16, one rounding of 2^-11."""
    x, weight, a, b, adapter, scale = make(5, 6, 7, 3, 2, dtype=HF)
    dy = torch.randn(5, 7, generator=torch.Generator().manual_seed(3)).to(HF).to(DEV)
    leaves = [t.detach().requires_grad_() for t in (x, weight, a, b)]
    got = torch.autograd.grad(lora.lora_linear(*leaves, adapter, scale), leaves, dy)
    points = [oracle.f64(t) for t in (x, weight, a, b)]

    def value():
        out = points[0] @ points[1]
        for t, i in enumerate(adapter.tolist()):
            if i >= 0:
                out[t] += float(scale[i]) * (points[0][t] @ points[2][i] @ points[3][i])
        return (out * oracle.f64(dy)).sum()

    for which in range(4):
        flat = points[which].view(-1)
        want = torch.empty_like(flat)
        for e in range(flat.numel()):
            at = float(flat[e])
            sides = []
            for h in (1e-3, -1e-3):
                flat[e] = at + h
                sides.append(value())
            flat[e] = at
            want[e] = (sides[0] - sides[1]) / 2e-3
        want = want.view(points[which].shape)
        oracle.assert_within(got[which], want, 2.0 ** -11 * want.abs() + 1e-5 * (1 + want.abs().max()), f"gradient {which}")


def test_expanded_gradient():
    x, weight, a, b, adapter, scale = make(40, 64, 64, 8, 3)
    leaf = a.detach().requires_grad_()
    one = torch.randn(1, 64, generator=torch.Generator().manual_seed(3)).to(BF).to(DEV).expand(40, 64)
    p, = torch.autograd.grad(lora.lora_linear(x, weight, leaf, b, adapter, scale), leaf, one)
    q, = torch.autograd.grad(lora.lora_linear(x, weight, leaf, b, adapter, scale), leaf, one.contiguous())
    assert torch.equal(p, q)
    lora.lora_linear(x, weight, leaf, b, adapter, scale).sum().backward()
    assert torch.isfinite(leaf.grad).all()


@pytest.mark.parametrize("T,K,N", [(0, 64, 32), (5, 0, 32), (100, 0, 32), (5, 64, 0), (100, 64, 0)])
def test_empty(T, K, N):
    x, weight, a, b, adapter, scale = make(T, K, N, 8, 3)
    leaves = [t.detach().requires_grad_() for t in (x, weight, a, b)]
    y = lora.lora_linear(*leaves, adapter, scale)
    assert torch.equal(y, torch.zeros(T, N, dtype=BF, device=DEV))
    for leaf, grad in zip(leaves, torch.autograd.grad(y, leaves, torch.ones_like(y))):
        assert grad.shape == leaf.shape and torch.equal(grad, torch.zeros_like(grad))


@pytest.mark.parametrize("T,K,N,R,L,pattern,lay", [(48, 4096, 8192, 16, 64, "mixed", "cols"), (1, 4096, 4096, 16, 8, "one", "rows"),
                                                   (2048, 2048, 4096, 64, 6, "requests", "rows")])
def test_sizes_of_served_projections(T, K, N, R, L, pattern, lay):
    gen = torch.Generator(device=DEV).manual_seed(T)
    rnd = lambda *shape: torch.randn(*shape, device=DEV, dtype=BF, generator=gen)
    turn = (lambda t: t.transpose(-2, -1)) if lay == "cols" else (lambda t: t)
    size = (lambda *s: (*s[:-2], s[-1], s[-2])) if lay == "cols" else (lambda *s: s)
    x, weight = rnd(T, K), turn(rnd(*size(K, N)).mul_(K ** -0.5))
    a, b = turn(rnd(*size(L, K, R)).mul_(K ** -0.5)), turn(rnd(*size(L, R, N)).mul_(R ** -0.5))
    _, _, _, _, adapter, scale = make(T, 8, 8, 8, L, pattern=pattern)
    got = lora.lora_linear(x, weight, a, b, adapter, scale)
    keep = sorted({0, T // 3, T // 2, T - 1})
    want, bound = oracle.lora_linear(x[keep], weight, a, b, adapter[keep], scale)
    oracle.assert_within(got[keep], want, bound + (oracle.UNIT[BF] * (oracle.f64(x[keep]) @ oracle.f64(weight)).abs() if T > 64 else 0))


def test_offsets_past_32_bits():
    """Rows of x that lie so far apart that the last of them begins more than 2^32 bytes behind the first."""
    T, K, N, R = 600, 64, 64, 8
    wide = torch.empty(T, 3700000, dtype=BF, device=DEV)      # 4.4 GB
    x, weight, a, b, adapter, scale = make(T, K, N, R, 3)
    apart = wide[:, 8:8 + K]
    apart.copy_(x)
    check(apart, weight, a, b, adapter, scale)
    dy = torch.randn(T, N, generator=torch.Generator().manual_seed(3)).to(BF).to(DEV)
    grads = []
    for rows in (x, apart):
        leaf = a.detach().requires_grad_()
        grads.append(torch.autograd.grad(lora.lora_linear(rows, weight, leaf, b, adapter, scale), leaf, dy)[0])
    assert torch.equal(*grads)


@pytest.mark.parametrize("T", [12, 100])
def test_on_another_stream_and_in_a_graph(T):
    x, weight, a, b, adapter, scale = make(T, 512, 256, 16, 6)
    want = lora.lora_linear(x, weight, a, b, adapter, scale)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = lora.lora_linear(x, weight, a, b, adapter, scale)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = lora.lora_linear(x, weight, a, b, adapter, scale)
    for seed in range(1, 4):
        x2, _, _, _, adapter2, _ = make(T, 512, 256, 16, 6, seed=seed)
        x.copy_(x2)
        adapter.copy_(adapter2)
        want = lora.lora_linear(x, weight, a, b, adapter, scale)
        held.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held, want)


def test_compiled_ops_agree():
    x, weight, a, b, adapter, scale = make(70, 128, 64, 8, 3)
    ops = torch.ops.grouped_mm_bf16_amd
    out, low = ops.lora(x, weight, a, b, adapter, scale, True)
    assert torch.equal(out, lora.lora_linear(x, weight, a, b, adapter, scale))
    adapter.clamp_(min=0)       # rows without an adapter leave their part of `low` as it was
    torch.library.opcheck(ops.lora, (x, weight, a, b, adapter, scale, True), test_utils=("test_schema", "test_faketensor"))
    dy = torch.ones(70, 64, dtype=BF, device=DEV)
    torch.library.opcheck(ops.lora_grad, (x, dy, low, low.new_empty(0), adapter, scale, a, b, True, True),
                          test_utils=("test_schema", "test_faketensor"))
