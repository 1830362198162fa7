"""The steps of an expert layer that is trained, on a real MI355X, forward and backward, against the formulas in 64 bits: sizes around the
kernels' shapes, odd ones and strides, types, one choice and many, infinite logits; gradients also against differences; the layer as a whole,
captured, on another stream."""
import pytest
import torch

from grouped_mm_bf16_amd import moe, moe_train
from oracle import operators_oracle as plain
from oracle import training_oracle as oracle

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF, SF = torch.bfloat16, torch.float16, torch.float32


def randn(gen, *shape, dtype=SF, pad=0):
    t = torch.randn(*shape[:-1], shape[-1] + pad, generator=gen).to(dtype).to(DEV)
    return t[..., :shape[-1]]


def routed(T, E, k, seed=0, dtype=SF, renormalize=True):
    gen = torch.Generator().manual_seed(seed)
    logits = randn(gen, T, E, dtype=dtype)
    return logits, moe_train.route(logits, k, renormalize)


# ------------------------------------------------------------------ rows
def check_rows(T, E, k, H, dtype, pad=0):
    gen = torch.Generator().manual_seed(T + H)
    _, routing = routed(T, E, k, T + H)
    x = randn(gen, T, H, dtype=dtype, pad=pad).requires_grad_()
    y = randn(gen, T * k, H, dtype=dtype, pad=pad).requires_grad_()
    weight = routing.slot_weight.clone().requires_grad_()
    routing = routing._replace(slot_weight=weight)
    back, grad = randn(gen, T * k, H, dtype=dtype, pad=pad), randn(gen, T, H, dtype=dtype, pad=pad)
    rows = moe_train.sort_rows(x, routing)
    assert torch.equal(rows.cpu(), oracle.sorted_rows(x, routing.token_rows))
    assert torch.equal(rows.detach(), x.detach()[routing.row_token.long()])
    dx, = torch.autograd.grad(rows, x, back)
    plain.assert_within(dx, *oracle.sum_rows(back, routing.token_rows, None, T), "dx")
    out = moe_train.combine_rows(y, routing, k)
    plain.assert_within(out, *oracle.sum_rows(y, routing.token_rows, weight, T), "out")
    dy, dw = torch.autograd.grad(out, (y, weight), grad, retain_graph=True)
    want = oracle.combine_backward(grad, y, routing.token_rows, weight)
    plain.assert_within(dy, *want[:2], "dy")
    plain.assert_within(dw, *want[2:], "dweight")
    assert torch.equal(torch.autograd.grad(out, y, grad, retain_graph=True)[0], dy)
    assert torch.equal(torch.autograd.grad(out, weight, grad)[0], dw)
    with torch.no_grad():
        assert torch.equal(moe_train.combine_rows(y, routing, k), out) and torch.equal(moe_train.sort_rows(x, routing), rows)


@pytest.mark.parametrize("H", [1, 3, 4, 7, 8, 9, 63, 64, 72, 130, 512, 520, 1031, 2048, 2056, 4100, 8200])
@pytest.mark.parametrize("dtype", [BF, HF, SF])
def test_widths(H, dtype):
    check_rows(13, 6, 3, H, dtype)


@pytest.mark.parametrize("T", [1, 2, 31, 257, 3000])
@pytest.mark.parametrize("E,k", [(4, 1), (60, 4), (128, 8), (40, 9), (64, 32)])
def test_tokens_and_choices(T, E, k):
    check_rows(T, E, k, 136, BF)


@pytest.mark.parametrize("dtype", [BF, SF])
@pytest.mark.parametrize("pad", [1, 5, 8])
def test_rows_that_lie_apart(pad, dtype):
    check_rows(40, 8, 2, 200, dtype, pad)
    check_rows(40, 8, 2, 201, dtype, pad)


def test_many_rows():
    check_rows(9000, 8, 2, 1024, BF)


def test_no_rows_and_no_columns():
    for T, H in ((0, 64), (5, 0)):
        logits = torch.randn(T, 6, device=DEV)
        routing = moe_train.route(logits.requires_grad_(), 2)
        x = torch.randn(T, H, device=DEV, dtype=BF, requires_grad=True)
        rows = moe_train.sort_rows(x, routing)
        out = moe_train.combine_rows(rows, routing, 2)
        assert rows.shape == (2 * T, H) and out.shape == (T, H)
        dx, dl = torch.autograd.grad(out, (x, logits), torch.ones_like(out))
        assert dx.shape == (T, H) and torch.equal(dl, torch.zeros_like(logits))


def test_a_turned_gradient_and_a_broadcast_one():
    """The upstream gradient comes as it comes: transposed, or one value for all."""
    _, routing = routed(12, 5, 2)
    y = torch.randn(24, 40, device=DEV, requires_grad=True)
    out = moe_train.combine_rows(y, routing, 2)
    for grad in (torch.randn(40, 12, device=DEV).t(), torch.ones((), device=DEV).expand(12, 40)):
        got, = torch.autograd.grad(out, y, grad, retain_graph=True)
        want, = torch.autograd.grad(out, y, grad.contiguous(), retain_graph=True)
        assert torch.equal(got, want)


def test_slots_without_a_row_take_no_part():
    """A row number outside the rows: nothing is read or written there."""
    gen = torch.Generator().manual_seed(0)
    _, routing = routed(9, 4, 2)
    rows = routing.token_rows.clone()
    rows[3], rows[10] = -1, 18
    odd = routing._replace(token_rows=rows)
    y, grad = randn(gen, 18, 40), randn(gen, 9, 40)
    weight = routing.slot_weight.clone()
    zero = weight.clone()
    zero[3] = zero[10] = 0
    assert torch.equal(moe_train.combine_rows(y, odd, 2), moe_train.combine_rows(y, routing._replace(slot_weight=zero), 2))
    w = weight.requires_grad_()
    dw, = torch.autograd.grad(moe_train.combine_rows(y, odd._replace(slot_weight=w), 2), w, grad)
    want, = torch.autograd.grad(moe_train.combine_rows(y, routing._replace(slot_weight=w), 2), w, grad)
    want[3] = want[10] = 0
    assert torch.equal(dw, want)


def test_a_value_that_is_no_number_stays_in_its_row():
    _, routing = routed(20, 6, 2)
    y = torch.randn(40, 64, device=DEV)
    y[7, 5] = float("nan")
    out = moe_train.combine_rows(y, routing, 2)
    token = int(routing.row_token[7])
    assert out.isnan().nonzero().tolist() == [[token, 5]]


# ------------------------------------------------------------------ routing
@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (7, 5, 5), (33, 64, 3), (100, 65, 8), (9, 1023, 32), (2000, 128, 8)])
@pytest.mark.parametrize("dtype", [BF, HF, SF])
@pytest.mark.parametrize("renormalize", [True, False])
def test_weights_gradient(T, E, k, dtype, renormalize):
    gen = torch.Generator().manual_seed(E)
    logits = (randn(gen, T, E) * 3).to(dtype).requires_grad_()
    routing = moe_train.route(logits, k, renormalize)
    assert all(torch.equal(p.detach(), q) for p, q in zip(routing, moe.moe_route(logits.detach(), k, renormalize)))
    assert routing.slot_weight.requires_grad and not routing.offs.requires_grad
    grad = randn(gen, T * k)
    got, = torch.autograd.grad(routing.slot_weight, logits, grad)
    assert got.dtype == dtype
    plain.assert_within(got, *oracle.route_backward(grad, routing.slot_expert, routing.slot_weight, logits, renormalize), "dlogits")


@pytest.mark.parametrize("renormalize", [True, False])
def test_infinite_logits(renormalize):
    """All weight in equal shares on what equals an infinite maximum: the derivative of those shares; nothing is NaN."""
    inf = float("inf")
    logits = torch.tensor([[0.0, inf, 1.0, inf, -inf], [-inf, 2.0, 1.0, -inf, 0.0], [-inf] * 5], device=DEV).requires_grad_()
    routing = moe_train.route(logits, 3, renormalize)
    grad = torch.randn(9, generator=torch.Generator().manual_seed(0)).to(DEV)
    got, = torch.autograd.grad(routing.slot_weight, logits, grad)
    plain.assert_within(got, *oracle.route_backward(grad, routing.slot_expert, routing.slot_weight, logits, renormalize))


def test_logits_that_lie_apart():
    wide = torch.randn(20, 30, device=DEV)
    for renormalize in (True, False):
        got, want = (torch.autograd.grad(moe_train.route(z, 4, renormalize).slot_weight, z, torch.arange(80.0, device=DEV))[0]
                     for z in (wide[:, :24].requires_grad_(), wide[:, :24].contiguous().requires_grad_()))
        assert torch.equal(got, want)


# ------------------------------------------------------------------ activation
def check_gated(rows, inner, kind, dtype, pad=0, scale=1.0):
    gen = torch.Generator().manual_seed(rows + inner)
    h = (randn(gen, rows, inner * (2 if kind == "swiglu" else 1), pad=pad) * scale).to(dtype)
    h = h.requires_grad_()
    grad = randn(gen, rows, inner, dtype=dtype, pad=pad)
    out = moe_train.gated(h, kind)
    plain.assert_within(out, *oracle.gated(h, kind), "out")
    dh, = torch.autograd.grad(out, h, grad)
    plain.assert_within(dh, *oracle.gated_backward(grad, h, kind), "dh")
    assert torch.equal(moe_train.gated(h.detach(), kind), out)


@pytest.mark.parametrize("inner", [1, 3, 4, 5, 8, 9, 64, 100, 768, 1031, 2048, 2056, 14336])
@pytest.mark.parametrize("kind", ["silu", "swiglu"])
@pytest.mark.parametrize("dtype", [BF, HF, SF])
def test_activation(inner, kind, dtype):
    check_gated(11, inner, kind, dtype)


@pytest.mark.parametrize("rows", [1, 2, 33, 1025, 20000])
@pytest.mark.parametrize("pad", [0, 1, 8])
def test_activation_rows(rows, pad):
    check_gated(rows, 72, "swiglu", BF, pad)
    check_gated(rows, 73, "silu", SF, pad)


@pytest.mark.parametrize("dtype", [BF, HF, SF])
def test_activation_of_large_values(dtype):
    """Far from zero e^-g is infinite, or nothing: the result is the gate or zero, the slope one or zero."""
    check_gated(30, 64, "swiglu", dtype, scale=60.0)
    check_gated(30, 64, "silu", dtype, scale=400.0)


def test_activation_agrees_with_the_one_of_the_forward_layer():
    h = torch.randn(50, 256, device=DEV, dtype=BF)
    for kind in ("silu", "swiglu"):
        a, b = moe_train.gated(h, kind).float(), moe.moe_activation(h, kind).float()
        assert ((a - b).abs() <= 2.0 ** -7 * b.abs()).all()       # both are rounded once: neighbours at most


def test_activation_of_nothing():
    for shape in ((0, 64), (7, 0)):
        h = torch.randn(*shape, device=DEV, dtype=BF, requires_grad=True)
        out = moe_train.gated(h)
        dh, = torch.autograd.grad(out, h, torch.ones_like(out))
        assert out.shape == (shape[0], shape[1] // 2) and dh.shape == shape


# ------------------------------------------------------------------ the layer
def layer(T, E, k, H, inner, kind, dtype, seed=0, logits=SF):
    gen = torch.Generator().manual_seed(seed)
    leaves = [randn(gen, T, H, dtype=dtype), randn(gen, T, E).to(logits), (randn(gen, E, H, inner * (2 if kind == "swiglu" else 1)) * H ** -0.5).to(dtype),
              (randn(gen, E, inner, H) * inner ** -0.5).to(dtype)]
    return [t.requires_grad_() for t in leaves], randn(gen, T, H, dtype=dtype)


def formula(leaves, k, kind, renormalize, chosen):
    """The layer in 64 bits, with torch's own derivatives, for a choice of experts."""
    x, z, up, down = (plain.f64(t).requires_grad_() for t in leaves)
    p = torch.softmax(z.gather(1, chosen), 1) if renormalize else torch.softmax(z, 1).gather(1, chosen)
    out = torch.zeros_like(x)
    for e in range(z.size(1)):
        token, j = (chosen == e).nonzero(as_tuple=True)
        h = x[token] @ up[e]
        inner = down.size(1)
        h = torch.nn.functional.silu(h) if kind == "silu" else torch.nn.functional.silu(h[:, :inner]) * h[:, inner:]
        out = out.index_add(0, token, p[token, j][:, None] * (h @ down[e]))
    return out, (x, z, up, down)


@pytest.mark.parametrize("kind", ["silu", "swiglu"])
@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("T,E,k,H,inner,dtype", [(1, 4, 2, 64, 32, BF), (50, 8, 2, 128, 64, HF), (300, 12, 3, 136, 72, BF), (37, 5, 5, 33, 17, SF), (700, 64, 6, 256, 64, SF)])
def test_layer(T, E, k, H, inner, dtype, kind, renormalize):
    """Four results are rounded on the way forward (2^-8 of bf16, 2^-11 of fp16), and each of them, the upstream gradients of the products among
    them, once on the way back: a gradient sees at most eight roundings, relative to its terms, whose sum it is of the size of."""
    leaves, grad = layer(T, E, k, H, inner, kind, dtype)
    out = moe_train.moe_train(*leaves, k, kind, renormalize)
    got = torch.autograd.grad(out, leaves, grad)
    chosen = moe.moe_route(leaves[1].detach(), k).slot_expert.cpu().long().reshape(T, k)
    want, inputs = formula(leaves, k, kind, renormalize, chosen)
    wanted = torch.autograd.grad(want, inputs, plain.f64(grad))
    unit = plain.UNIT[dtype] if dtype != SF else 2.0 ** -20      # fp32: sums of up to 700 terms one after the other
    assert (plain.f64(out) - want).norm() <= 4 * unit * want.norm()
    for name, p, q, leaf in zip(("x", "logits", "up", "down"), got, wanted, leaves):
        assert p.dtype == leaf.dtype and p.shape == leaf.shape
        assert (plain.f64(p) - q).norm() <= 8 * unit * q.norm() + 1e-12, name
    empty = [e for e in range(E) if not (chosen == e).any()]
    assert not got[2][empty].any() and not got[3][empty].any()


def test_layer_without_gradients_is_the_forward_layer():
    leaves, _ = layer(200, 8, 2, 128, 128, "swiglu", BF)
    with torch.no_grad():
        a, b = moe_train.moe_train(*leaves, 2).float(), moe.moe_forward(*leaves, 2).float()
    assert (a - b).norm() <= 2 * 2.0 ** -8 * b.norm()


def test_against_differences():
    """The derivative along a direction, of fp32 kernels: two steps of 2^-7 to either side leave a 2^-14th of the third derivative, and 2^-24
    of the values, 2^7 times as large, in the quotient."""
    leaves, grad = layer(40, 6, 2, 64, 48, "swiglu", SF)
    direction = [torch.randn(t.shape, generator=torch.Generator().manual_seed(i)).to(DEV) * (0.05 if i == 1 else 1.0) * t.detach().std() for i, t in enumerate(leaves)]
    grads = torch.autograd.grad(moe_train.moe_train(*leaves, 2), leaves, grad)
    chosen = moe.moe_route(leaves[1].detach(), 2).slot_expert
    for i, (leaf, step, g) in enumerate(zip(leaves, direction, grads)):
        values = []
        for sign in (1, -1):
            moved = [t.detach() + (sign * 2.0 ** -7 * step if j == i else 0) for j, t in enumerate(leaves)]
            assert torch.equal(moe.moe_route(moved[1], 2).slot_expert, chosen)
            values.append((plain.f64(moe_train.moe_train(*moved, 2)) * plain.f64(grad)).sum())
        slope = (values[0] - values[1]) * 64
        want = (plain.f64(g) * plain.f64(step)).sum()
        size = plain.f64(g).norm() * plain.f64(step).norm()
        assert abs(slope - want) <= 2e-3 * size, i


def test_captured_with_its_backward_pass_and_replayed():
    leaves, grad = layer(90, 8, 2, 128, 64, "swiglu", BF)
    run = lambda: (lambda out: (out.detach(), *torch.autograd.grad(out, leaves, grad)))(moe_train.moe_train(*leaves, 2))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = run()
    for seed in range(1, 4):
        others, grad2 = layer(90, 8, 2, 128, 64, "swiglu", BF, seed)
        with torch.no_grad():
            for p, q in zip(leaves, others):
                p.copy_(q)
            grad.copy_(grad2)
        want = run()
        for t in held:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(held, want))


def test_on_another_stream():
    leaves, grad = layer(64, 6, 2, 96, 64, "swiglu", BF)
    want = torch.autograd.grad(moe_train.moe_train(*leaves, 2), leaves, grad)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = torch.autograd.grad(moe_train.moe_train(*leaves, 2), leaves, grad)
    side.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(got, want))


@pytest.mark.parametrize("kind", ["silu", "swiglu"])
def test_compiled(kind):
    leaves, grad = layer(50, 6, 2, 128, 64, kind, BF)
    torch._dynamo.reset()
    results = []
    for f in (moe_train.moe_train, torch.compile(moe_train.moe_train, backend="aot_eager", fullgraph=True)):
        out = f(*leaves, 2, kind)
        results.append([out.detach(), *torch.autograd.grad(out, leaves, grad)])
        with torch.no_grad():
            results[-1].append(f(*leaves, 2, kind))
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(*results))


def test_pieces_compiled():
    leaves, _ = layer(50, 6, 3, 40, 64, "swiglu", SF)

    def pieces(x, z, up):
        routing = moe_train.route(z * 2, 3, False)
        return moe_train.combine_rows(moe_train.gated(moe_train.sort_rows(x * 2, routing), "swiglu") * 3, routing, 3) + up.sum()

    torch._dynamo.reset()
    results = []
    for f in (pieces, torch.compile(pieces, backend="aot_eager", fullgraph=True)):
        out = f(*leaves[:3])
        results.append([out.detach(), *torch.autograd.grad(out, leaves[:2], torch.ones_like(out))])
    assert all(torch.equal(p, q) for p, q in zip(*results))


def test_the_same_every_time():
    leaves, grad = layer(500, 16, 4, 256, 128, "swiglu", BF)
    first, again = (torch.autograd.grad(moe_train.moe_train(*leaves, 4), leaves, grad) for _ in range(2))
    assert all(torch.equal(p, q) for p, q in zip(first, again))
