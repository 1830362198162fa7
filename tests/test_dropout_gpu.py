"""Dropout on a real MI355X against its definition, the generator's bits among it: sizes around eight elements, strides, types, with and without a
residual, forward and backward; captured with a counter that is counted on."""
import pytest
import torch

from grouped_mm_bf16_amd import dropout as mod
from oracle import operators_oracle as plain
from oracle import training_oracle as oracle

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF, SF = torch.bfloat16, torch.float16, torch.float32
SEED, OFFSET = 0x123456789abcdef0, 0x0fedcba987654321


def rng(seed=SEED, offset=OFFSET):
    return torch.tensor([seed, offset], device=DEV)


def make(shape, dtype, pad=0, seed=0):
    gen = torch.Generator().manual_seed(seed)
    t = torch.randn(*shape[:-1], shape[-1] + pad, generator=gen).to(dtype).to(DEV)
    return t[..., :shape[-1]]


def check(shape, dtype, p=0.3, pad=0, residual=True, site=0, state=(SEED, OFFSET)):
    x, grad = make(shape, dtype, pad, 1).requires_grad_(), make(shape, dtype, pad, 2)
    other = make(shape, dtype, pad, 3).requires_grad_() if residual else None
    out = mod.dropout(x, p, rng(*state), other, site)
    want, bound, kept = oracle.dropout(x, p, *state, site, other)
    plain.assert_within(out, want, bound, "out")
    got = torch.autograd.grad(out, (x, other) if residual else (x,), grad)
    plain.assert_within(got[0], *oracle.dropout(grad, p, *state, site)[:2], "dx")
    assert torch.equal(got[0].cpu() != 0, kept & (grad.cpu() != 0))
    if residual:
        assert torch.equal(got[1], grad)
    with torch.no_grad():
        assert torch.equal(mod.dropout(x, p, rng(*state), other, site), out)
    return kept


@pytest.mark.parametrize("shape", [(1, 1), (1, 7), (1, 8), (3, 9), (5, 64), (7, 129), (2, 3, 40), (2, 5, 3, 11), (33,)])
@pytest.mark.parametrize("dtype", [BF, HF, SF])
@pytest.mark.parametrize("residual", [False, True])
def test_shapes(shape, dtype, residual):
    check(shape, dtype, residual=residual)


@pytest.mark.parametrize("pad", [1, 3, 8])
@pytest.mark.parametrize("width", [1, 5, 8, 24, 77])
@pytest.mark.parametrize("dtype", [BF, SF])
def test_rows_that_lie_apart(pad, width, dtype):
    kept = check((19, width), dtype, pad=pad)
    assert torch.equal(kept, check((19, width), dtype))


@pytest.mark.parametrize("p", [0.0, 2.0 ** -17, 2.0 ** -16, 0.1, 0.5, 0.999, 1.0])
def test_probabilities(p):
    kept = check((40, 100), SF, p)
    if p < 2.0 ** -16:
        assert kept.all()
    if p == 1.0:
        assert not kept.any()


@pytest.mark.parametrize("state", [(0, 0), (-1, -1), (1 << 40, 5), (7, -(1 << 63))])
@pytest.mark.parametrize("site", [0, 1, 65535])
def test_seeds_and_sites(state, site):
    check((6, 50), SF, 0.5, site=site, state=state)


def test_many_elements():
    """The share that is kept, to five deviations of it; blocks far into the counter against the definition."""
    x = torch.ones(3000, 4001, device=DEV)
    out = mod.dropout(x, 0.3, rng())
    n, p = x.numel(), round(0.3 * 65536) / 65536
    share = float((out != 0).double().mean())
    assert abs(share - (1 - p)) <= 5 * (p * (1 - p) / n) ** 0.5
    bits = oracle.dropout_bits(4096, SEED, OFFSET)
    assert torch.equal((out.reshape(-1)[:4096] != 0).cpu(), torch.from_numpy(bits >= round(0.3 * 65536)))
    other = mod.dropout(x, 0.3, rng(offset=OFFSET + 1))
    agree = float(((out != 0) == (other != 0)).double().mean())
    assert abs(agree - (p * p + (1 - p) ** 2)) <= 1e-3
    # the same elements of a type of another size, by other lanes
    assert torch.equal(mod.dropout(x.to(BF), 0.3, rng()) != 0, out != 0)


def test_what_is_dropped_counts_as_zero():
    """Infinities and NaN among it, forward and backward."""
    x = torch.full((8, 64), float("nan"), device=DEV)
    x[::2] = float("inf")
    kept = oracle.dropout(torch.ones(8, 64), 0.5, SEED, OFFSET)[2]
    x.requires_grad_()
    out = mod.dropout(x, 0.5, rng())
    assert torch.equal(out.cpu() == 0, ~kept)
    grad, = torch.autograd.grad(out, x, torch.full_like(x, float("inf")))
    assert torch.equal(grad.cpu() == 0, ~kept) and torch.equal(grad.isinf().cpu(), kept)


def test_counted_on_before_the_backward_pass():
    """The backward pass makes the forward pass's mask, whatever rng holds by then."""
    x = torch.ones(10, 100, device=DEV, requires_grad=True)
    state = rng()
    out = mod.dropout(x, 0.5, state)
    state[1] += 1
    grad, = torch.autograd.grad(out, x, torch.ones_like(x))
    assert torch.equal(grad, out.detach()) and not torch.equal(mod.dropout(x.detach(), 0.5, state), out.detach())


def test_captured_with_its_backward_pass_and_replayed():
    x = torch.randn(50, 72, device=DEV, dtype=BF).requires_grad_()
    other, grad, state = torch.randn_like(x.detach()), torch.randn_like(x.detach()), rng(3, 0)

    def step():
        out = mod.dropout(x, 0.25, state, other, 2)
        return out.detach(), torch.autograd.grad(out, x, grad)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
        state[1] += 1
    for i in range(4):
        state.copy_(rng(3, 10 + i))
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(held, want)) and state.tolist() == [3, 11 + i]


def test_turned_and_broadcast_tensors():
    x, other = torch.randn(30, 20, device=DEV).t(), torch.randn(30, device=DEV).expand(20, 30)
    assert torch.equal(mod.dropout(x, 0.5, rng(), other), mod.dropout(x.contiguous(), 0.5, rng(), other.contiguous()))
    leaf = x.contiguous().requires_grad_()
    out = mod.dropout(leaf, 0.5, rng())
    got, = torch.autograd.grad(out.sum(), leaf)        # the upstream gradient is one value
    assert torch.equal(got != 0, out != 0)


def test_nothing():
    for shape in ((0, 64), (5, 0), (0,)):
        x = torch.randn(*shape, device=DEV, requires_grad=True)
        out = mod.dropout(x, 0.5, rng(), torch.randn(*shape, device=DEV))
        grad, = torch.autograd.grad(out, x, torch.ones_like(out))
        assert out.shape == shape and grad.shape == shape


@pytest.mark.parametrize("shape", [(4, 6, 40), (24, 40)])
def test_compiled(shape):
    x, other = make(shape, BF).requires_grad_(), make(shape, BF, 0, 3).requires_grad_()
    state = rng()
    f = lambda a, b, s: mod.dropout(a * 2, 0.5, s, b, 1) + 1
    torch._dynamo.reset()
    results = []
    for g in (f, torch.compile(f, backend="aot_eager", fullgraph=True)):
        out = g(x, other, state)
        results.append([out.detach(), *torch.autograd.grad(out, (x, other), torch.ones_like(out))])
        with torch.no_grad():
            results[-1].append(g(x, other, state))
    assert all(torch.equal(p, q) for p, q in zip(*results))
