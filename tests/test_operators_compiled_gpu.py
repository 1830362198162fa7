"""torch.compile(fullgraph=True) of functions that call layer norm, the projection with adapters and the expert layer for a few tokens, on a
real MI355X: no graph break, and bit for bit what the eager calls return, forward and backward."""
import pytest
import torch

import test_lora_gpu
import test_moe_few_gpu
import test_norm_gpu
from grouped_mm_bf16_amd import lora, moe, norm

pytestmark = pytest.mark.gpu
BF, HF, DEV = torch.bfloat16, torch.float16, "cuda"


def compiled(f):
    torch._dynamo.reset()
    return torch.compile(f, backend="aot_eager", fullgraph=True)


def check(f, leaves, need, others=()):
    """f(*leaves, *others), and the gradients of those leaves that `need` names."""
    leaves = [None if t is None else t.detach().requires_grad_(n) for t, n in zip(leaves, need)]
    inputs = [t for t, n in zip(leaves, need) if n]
    results = []
    for g in (f, compiled(f)):
        y = g(*leaves, *others)
        dy = torch.randn(y.shape, generator=torch.Generator().manual_seed(0)).to(y.dtype).to(DEV)
        results.append([y.detach(), *(torch.autograd.grad(y, inputs, dy) if inputs else ())])
    torch.cuda.synchronize()
    for k, (p, q) in enumerate(zip(*results)):
        assert p.shape == q.shape and p.stride() == q.stride() and torch.equal(p, q), k


@pytest.mark.parametrize("need", [(False, False, False), (True, True, True), (True, False, False), (False, True, True)])
@pytest.mark.parametrize("rows", ["matrix", "batch", "apart", "turned"])
def test_layer_norm(need, rows):
    x, _, w, b = test_norm_gpu.make(24, 136, BF, BF, 1, pad=8 if rows == "apart" else 0)
    x = x.reshape(4, 6, 136) if rows in ("batch", "turned") else x
    x = x.transpose(0, 1) if rows == "turned" else x
    check(lambda x_, w_, b_: norm.layer_norm(x_ * 2, w_, b_) + 1, (x, w, b), need)
    check(lambda x_, w_, b_: norm.layer_norm(x_, w_, b_, 1e-3), (x, w, b), need)


def test_layer_norm_without_parameters():
    x, _, w, b = test_norm_gpu.make(24, 136, HF, torch.float32, 1)
    check(lambda x_, w_, b_: norm.layer_norm(x_, w_, b_), (x, None, b), (True, False, True))
    check(lambda x_: norm.layer_norm(x_), (x,), (True,))


@pytest.mark.parametrize("T", [20, 100, 400])
@pytest.mark.parametrize("need", [(False, False, False, False), (True, True, True, True), (True, False, True, True), (False, False, True, False),
                                  (True, False, False, False), (False, False, False, True)])
@pytest.mark.parametrize("lay", ["rows", "cols"])
def test_adapters(T, need, lay):
    x, weight, a, b, adapter, scale = test_lora_gpu.make(T, 264, 136, 8, 3, lay)
    check(lambda x_, w_, a_, b_, at, s: lora.lora_linear(x_ * 2, w_, a_, b_, at, s) + 1, (x, weight, a, b), need, (adapter, scale))
    check(lambda x_, w_, a_, b_, at: lora.lora_linear(x_, w_, a_, b_, at), (x, weight, a, b), need, (adapter,))


@pytest.mark.parametrize("kind", ["silu", "swiglu", "interleaved"])
@pytest.mark.parametrize("T", [1, 20, 64])
def test_expert_layer(kind, T):
    x, z, up, down = test_moe_few_gpu.make(T, 6, 136, 128, kind)
    check(lambda *t: test_moe_few_gpu.run(*t, 2, kind) * 2, (x, z, up, down), (False,) * 4)


def test_a_block_of_them():
    x, weight, a, b, adapter, scale = test_lora_gpu.make(40, 128, 128, 8, 3)
    _, z, up, down = test_moe_few_gpu.make(40, 6, 128, 64)

    def block(x_, w_, a_, b_, z_, up_, down_, at, s):
        h = x_ + lora.lora_linear(norm.layer_norm(x_), w_, a_, b_, at, s)
        return h + moe.moe_forward_few(norm.layer_norm(h), z_, up_, down_, 2)

    check(block, (x, weight, a, b, z, up, down), (False,) * 7, (adapter, scale))
