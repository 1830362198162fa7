"""A block of the package's operators run together, on a real MI355X: against the formula in 64 bits, replayed from a graph, and tuned."""
import pytest
import torch

from grouped_mm_bf16_amd import expert_block
from oracle import operators_oracle as oracle

pytestmark = pytest.mark.gpu
DEV = "cuda"


def small(seed=0):
    block = expert_block.random_block(256, 12, 3, 128, 5, 8, device=DEV, seed=seed)
    block.lora_b.copy_(torch.randn(block.lora_b.shape, generator=torch.Generator().manual_seed(seed)).mul_(0.3))
    return block


def batch(T, seed=0):
    gen = torch.Generator().manual_seed(100 + seed + T)
    return (torch.randn(T, 256, generator=gen).to(torch.bfloat16).to(DEV),
            torch.randint(-1, 5, (T,), generator=gen).to(torch.int32).to(DEV))


@pytest.mark.parametrize("T", [1, 7, 64, 65, 200])
def test_against_the_formula(T):
    """Each of the seven operations rounds its result to bf16 (2^-8 of it): of the block's result, whose parts are of its own size, seven
    of those (the choice of the experts is taken from the run itself: two logits that nearly tie may change places)."""
    block, (x, adapter) = small(), batch(T)
    got = block(x, adapter)
    h = oracle.f64(x) + oracle.lora_linear(oracle.layer_norm(x, *block.norm_in), block.projection, block.lora_a, block.lora_b, adapter,
                                           block.scale, torch.bfloat16)[0]
    run_h = block.project(x, adapter)
    assert (oracle.f64(run_h) - h).norm() <= 3 * 2.0 ** -8 * h.norm()
    n = expert_block.norm.layer_norm(run_h, *block.norm_experts)
    logits = expert_block.grouped_mm(n.unsqueeze(0), block.router.unsqueeze(0)).squeeze(0)
    y, _ = oracle.moe_layer(n, logits.cpu(), block.w_up.cpu(), block.w_down.cpu(), block.top_k, "swiglu")
    want = oracle.f64(run_h) + y
    assert (oracle.f64(got) - want).norm() <= 5 * 2.0 ** -8 * want.norm()


def test_replayed_from_a_graph():
    block, (x, adapter) = small(), batch(16)
    block(x, adapter)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = block(x, adapter)
    for seed in range(1, 4):
        x2, adapter2 = batch(16, seed)
        x.copy_(x2)
        adapter.copy_(adapter2)
        want = block(x, adapter)
        held.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held, want)


def test_a_tuning_step_is_the_formulas():
    """A step of gradient descent on the adapters, B then A seen through a rounding of 2^-8 each (the gradient, the step, the parameter), the
    error's gradient through one of the projection's result (2^-8 of its terms)."""
    block, (x, adapter) = small(), batch(300)
    target = torch.randn(300, 256, generator=torch.Generator().manual_seed(7)).to(torch.bfloat16).to(DEV)
    before = [oracle.f64(t) for t in (block.lora_a, block.lora_b)]
    normed = oracle.layer_norm(x, *block.norm_in)
    out = oracle.f64(x) + oracle.lora_linear(normed, block.projection, block.lora_a, block.lora_b, adapter, block.scale, torch.bfloat16)[0]
    off = out - oracle.f64(target)
    dy = 2 * off / off.numel()
    (_, _, (da, _), (db, _)) = oracle.lora_backward(dy, normed, block.projection, block.lora_a, block.lora_b, adapter, block.scale, torch.bfloat16)
    losses = expert_block.tune(block, x, adapter, target, 1, 0.5)
    assert len(losses) == 1 and abs(losses[0] - float(off.square().mean())) <= 2.0 ** -6 * float(off.square().mean())
    for p, old, grad in zip((block.lora_a, block.lora_b), before, (da, db)):
        want = old - 0.5 * grad
        assert (oracle.f64(p) - want).norm() <= 2.0 ** -8 * want.norm() + 8 * 2.0 ** -8 * (0.5 * grad).norm()
    for i in range(5):
        if not (adapter == i).any():
            assert torch.equal(oracle.f64(block.lora_b[i]), before[1][i])
