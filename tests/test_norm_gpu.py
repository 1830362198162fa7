"""Layer norm on a real MI355X, forward and backward, against the formulas in 64 bits: widths around the kernels' shapes, odd sizes and
strides, types of rows and parameters, few and many rows; gradients also against differences."""
import pytest
import torch

from grouped_mm_bf16_amd import norm
from oracle import operators_oracle as oracle

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF, SF = torch.bfloat16, torch.float16, torch.float32


def make(rows, width, dtype, param_dtype, seed, pad=0, offset=0):
    gen = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, width + pad + offset, generator=gen) * 2 + 0.5).to(dtype).to(DEV)[:, offset:offset + width]
    dy = torch.randn(rows, width + pad + offset, generator=gen).to(dtype).to(DEV)[:, offset:offset + width]
    w = (1 + 0.2 * torch.randn(width, generator=gen)).to(param_dtype).to(DEV)
    b = (0.2 * torch.randn(width, generator=gen)).to(param_dtype).to(DEV)
    return x, dy, w, b


def check(x, dy, w, b, eps=1e-5):
    param_dtype = w.dtype if w is not None else x.dtype
    leaves = [None if t is None else t.detach().requires_grad_() for t in (x, w, b)]
    y = norm.layer_norm(*leaves, eps)
    given = [t for t in leaves if t is not None]
    grads = iter(torch.autograd.grad(y, given, dy))
    plain = norm.layer_norm(x, w, b, eps)
    assert torch.equal(plain, y), "with and without a graph"
    assert y.dtype == x.dtype and y.shape == x.shape
    bounds = oracle.layer_norm_bounds(dy, x, w, b, eps, x.dtype, param_dtype)
    oracle.assert_within(y, oracle.layer_norm(x, w, b, eps), bounds[0], "y")
    want = oracle.layer_norm_backward(dy, x, w, eps)
    for name, leaf, value, bound in zip(("dx", "dweight", "dbias"), leaves, want, bounds[1:]):
        if leaf is not None:
            got = next(grads)
            assert got.dtype == leaf.dtype and got.shape == leaf.shape
            oracle.assert_within(got, value, bound, name)


@pytest.mark.parametrize("width", [1, 2, 7, 8, 63, 64, 65, 128, 200, 256, 257, 512, 520, 1024, 1031, 2048, 2056, 4096, 4100, 8192,
                                   8200, 16383, 16384])
@pytest.mark.parametrize("dtype", [BF, HF, SF])
def test_widths(width, dtype):
    check(*make(9, width, dtype, dtype, width))


@pytest.mark.parametrize("rows", [1, 2, 3, 31, 33, 512, 513, 1100, 3001])
@pytest.mark.parametrize("width", [64, 136, 1000, 2304])
def test_rows(rows, width):
    check(*make(rows, width, BF, BF, rows + width))


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("width", [96, 1031, 4096])
def test_parameters_in_float32(width, dtype):
    check(*make(130, width, dtype, SF, width))


@pytest.mark.parametrize("pad,offset", [(8, 0), (3, 0), (0, 1), (8, 8), (5, 3)])
@pytest.mark.parametrize("dtype", [BF, SF])
def test_rows_that_lie_apart(pad, offset, dtype):
    check(*make(70, 768, dtype, dtype, pad + offset, pad, offset))


@pytest.mark.parametrize("with_weight,with_bias", [(False, False), (True, False), (False, True)])
def test_without_parameters(with_weight, with_bias):
    x, dy, w, b = make(40, 1000, BF, BF, 5)
    check(x, dy, w if with_weight else None, b if with_bias else None)


def test_constant_rows_and_large_means():
    """A variance of zero leaves eps alone; a mean far from zero must not eat the variance (two sums, not the sum of squares)."""
    gen = torch.Generator().manual_seed(0)
    x = torch.full((4, 512), 3.0)
    x[1] = 0.0
    x[2] = 4096.0 + torch.randn(512, generator=gen)
    x[3] = -1e4
    x, dy = x.to(DEV), torch.randn(4, 512, generator=gen).to(DEV)
    w = torch.ones(512, device=DEV)
    check(x, dy, w, torch.zeros(512, device=DEV))


def test_nan_and_infinity_stay_in_their_rows():
    x, dy, w, b = make(6, 300, BF, BF, 1)
    x[1, 5], x[4, 299] = float("nan"), float("inf")
    y = norm.layer_norm(x, w, b)
    good = [0, 2, 3, 5]
    assert y[[1, 4]].isnan().all() and torch.isfinite(y[good]).all()
    assert torch.equal(y[good], norm.layer_norm(x[good], w, b))


def test_each_gradient_alone_and_the_same_every_time():
    x, dy, w, b = make(700, 1152, BF, BF, 3)
    leaves = [t.detach().requires_grad_() for t in (x, w, b)]
    every = torch.autograd.grad(norm.layer_norm(*leaves), leaves, dy)
    for i in range(3):
        alone = [t.detach() for t in (x, w, b)]
        alone[i].requires_grad_()
        assert torch.equal(torch.autograd.grad(norm.layer_norm(*alone), alone[i], dy)[0], every[i])


def test_gradients_against_differences():
    """Central differences of the formula in 64 bits, step 1e-4: their error is of the order of 1e-8; fp32 arithmetic 1e-5."""
    x, dy, w, b = make(3, 40, SF, SF, 11)
    leaves = [t.detach().requires_grad_() for t in (x, w, b)]
    got = torch.autograd.grad(norm.layer_norm(*leaves), leaves, dy)
    points = [oracle.f64(t) for t in (x, w, b)]
    weigh = oracle.f64(dy)
    for which in range(3):
        flat = points[which].view(-1)
        want = torch.empty_like(flat)
        for i in range(flat.numel()):
            at = float(flat[i])
            sides = []
            for h in (1e-4, -1e-4):
                flat[i] = at + h
                sides.append((oracle.layer_norm(*points) * weigh).sum())
            flat[i] = at
            want[i] = (sides[0] - sides[1]) / 2e-4
        oracle.assert_within(got[which], want.view(points[which].shape), 2e-5 * (1 + want.abs().max()), f"gradient {which}")


def test_other_shapes_and_empty_tensors():
    gen = torch.Generator().manual_seed(2)
    x = torch.randn(3, 5, 7, 48, generator=gen).to(BF).to(DEV)
    w = torch.ones(48, device=DEV, dtype=BF)
    flat = norm.layer_norm(x.reshape(-1, 48), w)
    assert torch.equal(norm.layer_norm(x, w).reshape(-1, 48), flat)
    turned = norm.layer_norm(x.transpose(0, 2), w)
    assert torch.equal(turned.transpose(0, 2).reshape(-1, 48), flat)
    assert torch.equal(norm.layer_norm(x[0, 0, 0], w), flat[0])
    for shape in ((0, 48), (4, 0), (0, 0)):
        e = torch.empty(shape, device=DEV, dtype=BF, requires_grad=True)
        p = torch.ones(shape[1], device=DEV, dtype=BF, requires_grad=True)
        y = norm.layer_norm(e, p)
        ge, gp = torch.autograd.grad(y, (e, p), torch.empty_like(y))
        assert y.shape == e.shape == ge.shape and torch.equal(gp, torch.zeros_like(p))


def test_gradient_that_is_expanded():
    x, dy, w, b = make(20, 256, BF, BF, 9)
    leaf = x.detach().requires_grad_()
    one = dy[:1].expand(20, 256)
    a, = torch.autograd.grad(norm.layer_norm(leaf, w, b), leaf, one)
    c, = torch.autograd.grad(norm.layer_norm(leaf, w, b), leaf, one.contiguous())
    assert torch.equal(a, c)
    norm.layer_norm(leaf, w, b).sum().backward()     # a gradient of stride 0 in both dimensions
    assert torch.isfinite(leaf.grad).all()


def test_on_another_stream_and_in_a_graph():
    x, dy, w, b = make(64, 1024, BF, BF, 4)
    want = norm.layer_norm(x, w, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = norm.layer_norm(x, w, b)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = norm.layer_norm(x, w, b)
    for k in range(3):
        x.copy_(make(64, 1024, BF, BF, 20 + k)[0])
        want = norm.layer_norm(x, w, b)
        held.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held, want)


def test_compiled_ops_agree():
    x, dy, w, b = make(10, 264, BF, BF, 6)
    out, stats = torch.ops.grouped_mm_bf16_amd.layer_norm(x, w, b, 1e-5, True)
    assert torch.equal(out, norm.layer_norm(x, w, b))
    torch.library.opcheck(torch.ops.grouped_mm_bf16_amd.layer_norm, (x, w, b, 1e-5, True), test_utils=("test_schema", "test_faketensor"))
    torch.library.opcheck(torch.ops.grouped_mm_bf16_amd.layer_norm_backward, (dy, x, w, stats, BF, True, True, True),
                          test_utils=("test_schema", "test_faketensor"))
