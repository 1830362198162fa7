"""The block of the package's operators as it is trained and with 8-bit weights, on a real MI355X: against the formulas in 64 bits, forward and
backward; replayed from graphs; its operators compiled together."""
import pytest
import torch

import test_expert_block_gpu as common
from grouped_mm_bf16_amd import dropout, expert_block, int8, lora, moe, moe_train, norm
from oracle import int8_oracle, operators_oracle as plain, training_oracle

pytestmark = pytest.mark.gpu
DEV = "cuda"
UNIT = 2.0 ** -8


def counter(seed=11, offset=5):
    return torch.tensor([seed, offset], device=DEV)


def masks(T, p, rng, site=0):
    limit, (seed, offset) = round(p * 65536), rng.tolist()
    return [torch.from_numpy(training_oracle.dropout_bits(T * 256, seed, offset, site + i) >= limit).reshape(T, 256) * (65536 / (65536 - limit)) for i in range(2)]


def formula(x, weights, scale, top_k, adapter, kept, chosen):
    """The trained block on 64-bit leaves, for the experts that were chosen."""
    w_in, b_in, projection, lora_a, lora_b, w_ex, b_ex, router, up, down = weights
    n = torch.nn.functional.layer_norm(x, (x.size(1),), w_in, b_in)
    low = torch.stack([n[t] @ projection + (scale[i] * (n[t] @ lora_a[i]) @ lora_b[i] if i >= 0 else 0) for t, i in enumerate(adapter.tolist())])
    h = x + low * kept[0]
    n = torch.nn.functional.layer_norm(h, (x.size(1),), w_ex, b_ex)
    weight = torch.softmax((n @ router).gather(1, chosen), 1)
    out = torch.zeros_like(x)
    for e in chosen.unique().tolist():
        token, j = (chosen == e).nonzero(as_tuple=True)
        g, u = (n[token] @ up[e]).chunk(2, 1)
        out = out.index_add(0, token, weight[token, j][:, None] * ((torch.nn.functional.silu(g) * u) @ down[e]))
    return h + out * kept[1]


def choice(block, x, adapter, p, rng):
    """Of the run itself: two logits that nearly tie may change places."""
    with torch.no_grad():
        low = lora.lora_linear(norm.layer_norm(x, *block.norm_in), block.projection, block.lora_a, block.lora_b, adapter, block.scale)
        n = norm.layer_norm(dropout.dropout(low, p, rng, x), *block.norm_experts)
        logits = expert_block._logits(n, block.router)
        return moe.moe_route(logits, block.top_k).slot_expert.cpu().long().reshape(x.size(0), -1)


@pytest.mark.parametrize("p", [0.0, 0.25])
@pytest.mark.parametrize("T", [1, 7, 65, 200])
def test_training_against_the_formula(T, p):
    """A value has seen at most twelve roundings on its way forward (norms, the adapter's two products, two sums, the logits, the experts' four, their
    weights' logits), a gradient as many again on its way back."""
    block, (x, adapter) = common.small(), common.batch(T)
    rng = counter()
    leaves = [x.requires_grad_(), *(t.requires_grad_() for t in block.weights())]
    grad = torch.randn(T, 256, generator=torch.Generator().manual_seed(T)).to(torch.bfloat16).to(DEV)
    out = block.train(x, adapter, p, rng)
    got = torch.autograd.grad(out, leaves, grad)
    inputs = [plain.f64(t).requires_grad_() for t in leaves]
    want = formula(inputs[0], inputs[1:], plain.f64(block.scale), block.top_k, adapter, masks(T, p, rng), choice(block, x, adapter, p, rng))
    wanted = torch.autograd.grad(want, inputs, plain.f64(grad))
    assert (plain.f64(out) - want).norm() <= 12 * UNIT * want.norm()
    for i, (g, w, leaf) in enumerate(zip(got, wanted, leaves)):
        assert g.shape == leaf.shape and g.dtype == leaf.dtype
        assert (plain.f64(g) - w).norm() <= 24 * UNIT * w.norm(), i


def test_without_dropout_it_is_the_block():
    block, (x, adapter) = common.small(), common.batch(90)
    with torch.no_grad():
        a, b = plain.f64(block.train(x, adapter, 0.0, counter())), plain.f64(block(x, adapter))
    # the experts' sum of either has seen up to five roundings, the block's two
    assert (a - b).norm() <= 2 * 7 * UNIT * b.norm()


def test_training_replayed_from_a_graph():
    """The counter is counted on in the graph: every replay has masks of its own."""
    block, (x, adapter) = common.small(), common.batch(40)
    weights = [t.requires_grad_() for t in block.weights()]
    rng, grad = counter(), torch.ones_like(x)

    def run():
        out = block.train(x, adapter, 0.25, rng)
        result = (out.detach(), *torch.autograd.grad(out, weights, grad))
        rng[1].add_(1)
        return result

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = run()
    for seed in range(1, 4):
        x2, adapter2 = common.batch(40, seed)
        x.copy_(x2)
        adapter.copy_(adapter2)
        before = rng.clone()
        want = run()
        after = rng.clone()
        rng.copy_(before)
        for t in held:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(rng, after) and all(torch.equal(p, q) for p, q in zip(held, want))
        graph.replay()      # the next masks
        torch.cuda.synchronize()
        assert not torch.equal(held[0], want[0])


def test_training_steps_run():
    block, (x, adapter) = common.small(), common.batch(120)
    target = torch.randn(120, 256, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16).to(DEV)
    before = [t.clone() for t in block.weights()]
    out = plain.f64(block.train(x, adapter, 0.1, torch.tensor([4, 0], device=DEV)))
    losses = expert_block.train(block, x, adapter, target, 2, 0.0, seed=4)
    assert len(losses) == 2 and losses[0] != losses[1]      # other masks
    want = float((out - plain.f64(target)).square().mean())
    assert abs(losses[0] - want) <= 1e-4 * want              # sums of 2^15 squares in fp32
    assert all(torch.equal(p, q) for p, q in zip(before, block.weights()))
    expert_block.train(block, x, adapter, target, 1, 1.0, seed=4)
    assert all(not torch.equal(p, q) for p, q in zip(before, block.weights()))


# ------------------------------------------------------------------ 8-bit weights
@pytest.mark.parametrize("adapter", [-1, 2])
@pytest.mark.parametrize("T", [1, 7, 64, 65, 200])
def test_eight_bit_against_the_formula(T, adapter):
    """Of the first half two roundings to bf16; of the second the logits' apart (the choice and the norm are the run's own), the experts' two and
    the activations' steps as for the layer alone, and the sum's."""
    block, (x, _) = common.small(), common.batch(T)
    eight = block.eight_bit(adapter)
    got = eight(x)
    merged = plain.f64(block.projection)
    if adapter >= 0:
        merged = merged + plain.f64(block.scale)[adapter] * (plain.f64(block.lora_a[adapter]) @ plain.f64(block.lora_b[adapter]))
    values, scale = plain.f64(eight.projection.values), plain.f64(eight.projection.scale)
    # half a step; 16 roundings of fp32 of sums that are no larger than 127 steps leave less than a 1000th of one
    assert ((values * scale - merged).abs() <= 0.501 * scale).all()
    normed = norm.layer_norm(x, *block.norm_in)
    q, s = int8_oracle.quantize(normed)
    h = plain.f64(x) + int8_oracle.mm(q, s, eight.projection.values, eight.projection.scale, torch.bfloat16)[0]
    run_h = x + int8.linear_int8(normed, eight.projection)
    assert (plain.f64(run_h) - h).norm() <= 2 * UNIT * h.norm()
    n = norm.layer_norm(run_h, *block.norm_experts)
    logits = expert_block._logits(n, block.router)
    y = int8_oracle.layer(n, logits, eight.w_up.values, eight.w_up.scale, eight.w_down.values, eight.w_down.scale, block.top_k, "swiglu")
    want = plain.f64(run_h) + y
    assert (plain.f64(got) - want).norm() <= 5 * UNIT * want.norm()
    full = plain.f64(block(x, torch.full((T,), adapter, dtype=torch.int32, device=DEV)))
    # half a step of either operand at random, 3 of 100 of a product (of linear layers and experts both), and experts that nearly tie
    if T >= 64:
        assert (plain.f64(got) - full).norm() <= 0.15 * full.norm()


def test_eight_bit_replayed_from_a_graph():
    block, (x, _) = common.small(), common.batch(5)
    eight = block.eight_bit()
    eight(x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = eight(x)
    for seed in range(1, 4):
        x.copy_(common.batch(5, seed)[0])
        want = eight(x)
        held.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held, want)


# ------------------------------------------------------------------ compiled
def test_compiled_together():
    block, (x, adapter) = common.small(), common.batch(70)
    eight, rng = block.eight_bit(), counter()

    def training(x_, w_, a_, b_, router, up, down):
        h = dropout.dropout(lora.lora_linear(norm.layer_norm(x_), w_, a_, b_, adapter, block.scale), 0.25, rng, x_)
        n = norm.layer_norm(h)
        return dropout.dropout(moe_train.moe_train(n, n @ router, up, down, 3), 0.25, rng, h, 1)

    leaves = [t.detach().requires_grad_() for t in (x, block.projection, block.lora_a, block.lora_b, block.router, block.w_up, block.w_down)]
    torch._dynamo.reset()
    results = []
    for f in (training, torch.compile(training, backend="aot_eager", fullgraph=True)):
        out = f(*leaves)
        results.append([out.detach(), *torch.autograd.grad(out, leaves, torch.ones_like(out))])

    def serving(x_):
        h = x_ + int8.linear_int8(norm.layer_norm(x_), eight.projection)
        n = norm.layer_norm(h)
        return h + int8.moe_forward_int8(n, n @ eight.router, eight.w_up, eight.w_down, 3)

    with torch.no_grad():
        for rows in (x.detach(), x.detach()[:3]):
            for r, f in zip(results, (serving, torch.compile(serving, backend="aot_eager", fullgraph=True))):
                r.append(f(rows))
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(*results))
