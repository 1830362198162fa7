"""What torch would differentiate that has no derivative here raises (CPU: the kernels are replaced by the formulas, without a graph)."""
import pytest
import torch
from torch.autograd import forward_ad

from grouped_mm_bf16_amd import api, expert_block, kernels, lora, moe, norm


@pytest.fixture
def formulas(monkeypatch):
    """The launches, as opaque to torch as they are."""
    def norm_forward(x, weight, bias, eps, save):
        with torch.no_grad():
            mean = x.mean(1)
            rstd = 1 / ((x - mean[:, None]).square().mean(1) + eps).sqrt()
            y = (x - mean[:, None]) * rstd[:, None] * (1 if weight is None else weight) + (0 if bias is None else bias)
            return y, torch.stack([mean, rstd]) if save else None

    def norm_backward(dy, x, weight, stats, param_dtype, need_x, need_weight, need_bias):
        with torch.no_grad():
            z = (x - stats[0][:, None]) * stats[1][:, None]
            g = dy * (1 if weight is None else weight)
            dx = stats[1][:, None] * (g - g.mean(1, keepdim=True) - z * (g * z).mean(1, keepdim=True))
            return [dx, (dy * z).sum(0), dy.sum(0)]

    def per_token(x, a, b, adapter, scale):
        return torch.stack([float(scale[i]) * (x[t] @ a[i]) @ b[i] for t, i in enumerate(adapter.tolist())])

    def lora_forward(x, weight, a, b, adapter, scale, save):
        with torch.no_grad():
            low = torch.stack([x[t] @ a[i] for t, i in enumerate(adapter.tolist())])
            return x @ weight + per_token(x, a, b, adapter, scale), low if save else None

    def lora_grad(x, dy, low, u, adapter, scale, a, b, need_a, need_b):
        with torch.no_grad():
            da, db = torch.zeros_like(a), torch.zeros_like(b)
            for t, i in enumerate(adapter.tolist()):
                da[i] += float(scale[i]) * torch.outer(x[t], b[i] @ dy[t])
                db[i] += float(scale[i]) * torch.outer(low[t], dy[t])
            return [da, db]

    for module, name, to in ((norm, "_require_gpu", lambda *t: None), (lora, "_require_gpu", lambda *t: None),
                             (norm, "_forward_now", norm_forward), (norm, "_backward_now", norm_backward),
                             (lora, "_forward_now", lora_forward), (lora, "_grad_now", lora_grad),
                             (kernels, "grouped_mm_3d3d", lambda p, q, out: out.copy_(p @ q))):
        monkeypatch.setattr(module, name, to)


def norm_call(seed=0):
    gen = torch.Generator().manual_seed(seed)
    leaves = [torch.randn(5, 8, generator=gen), torch.randn(8, generator=gen), torch.randn(8, generator=gen)]
    return norm.layer_norm, leaves, lambda x, w, b: torch.nn.functional.layer_norm(x, (8,), w, b)


def lora_call(seed=0):
    gen = torch.Generator().manual_seed(seed)
    leaves = [torch.randn(*s, generator=gen).to(torch.float16) for s in ((5, 6), (6, 7), (3, 6, 2), (3, 2, 7))]
    adapter, scale = torch.tensor([0, 2, 2, 1, 0], dtype=torch.int32), torch.ones(3)
    return lambda *t: lora.lora_linear(*t, adapter, scale), leaves, None


CALLS = pytest.mark.parametrize("call", [norm_call, lora_call])


@CALLS
def test_first_derivatives(formulas, call):
    """The same with and without create_graph."""
    f, leaves, plain = call()
    leaves = [t.requires_grad_() for t in leaves]
    y = f(*leaves)
    dy = torch.ones_like(y)
    grads = torch.autograd.grad(y, leaves, dy, retain_graph=True)
    again = torch.autograd.grad(y, leaves, dy, create_graph=True)
    for i, (p, q) in enumerate(zip(grads, again)):
        assert torch.equal(p, q.detach()) and not p.requires_grad
        if plain:
            want = torch.autograd.grad(plain(*leaves), leaves, dy)
            assert torch.allclose(p, want[i], atol=1e-5)


@CALLS
@pytest.mark.parametrize("through", ["sum", "cubes"])
def test_second_derivatives_raise(formulas, call, through):
    """A gradient penalty, for an upstream gradient that requires a gradient itself (cubes) and for a constant one."""
    for which in range(3):
        f, leaves, _ = call()
        leaves[which].requires_grad_()
        leaf = leaves[which]
        y = f(*leaves)
        value = y.float().sum() if through == "sum" else (y.float() ** 3).sum()
        grad, = torch.autograd.grad(value, leaf, create_graph=True)
        with pytest.raises(RuntimeError, match="no second derivative"):
            (value + grad.float().square().sum()).backward()


def test_second_derivatives_raise_for_copied_operands(formulas):
    """The saved rows are a copy, which has no graph of its own."""
    x = torch.randn(4, 6, 8).transpose(0, 1).requires_grad_()
    y = norm.layer_norm(x)
    grad, = torch.autograd.grad(y.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="no second derivative"):
        grad.square().sum().backward()


@CALLS
@pytest.mark.parametrize("which", [0, 1, 2])
def test_forward_mode_raises(formulas, call, which):
    f, leaves, _ = call()
    plain = f(*leaves)
    with forward_ad.dual_level():
        assert torch.equal(f(*leaves), plain)       # no tangent: as ever
        leaves[which] = forward_ad.make_dual(leaves[which], torch.ones_like(leaves[which]))
        with pytest.raises(NotImplementedError, match="jvp"):
            f(*leaves)
        with torch.no_grad(), pytest.raises(NotImplementedError, match="jvp"):
            f(*leaves)


@CALLS
def test_function_transforms_raise(formulas, call):
    f, leaves, _ = call()
    with pytest.raises((RuntimeError, NotImplementedError)):
        torch.func.jvp(f, tuple(leaves), tuple(torch.ones_like(t) for t in leaves))


# ------------------------------------------------------------------ forward only
def layer_args():
    bf = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)
    return [bf(4, 64), torch.zeros(4, 8), bf(8, 64, 64), bf(8, 32, 64)]


@pytest.fixture
def few_launched(monkeypatch):
    launched = []
    monkeypatch.setattr(moe, "_require_gpu", lambda *t: None)
    monkeypatch.setattr(moe, "_few_now", lambda x, *rest: launched.append(1) or torch.zeros_like(x))
    return launched


@pytest.mark.parametrize("which", range(4))
def test_few_tokens_refuse_a_gradient(few_launched, which):
    args = layer_args()
    args[which].requires_grad_()
    with pytest.raises(RuntimeError, match="forward only"):
        moe.moe_forward_few(*args, 2)
    assert not few_launched
    with torch.no_grad():
        assert not moe.moe_forward_few(*args, 2).requires_grad
    assert not moe.moe_forward_few(*(t.detach() for t in args), 2).requires_grad
    assert len(few_launched) == 2


@pytest.mark.parametrize("which", range(4))
def test_few_tokens_refuse_a_tangent(few_launched, which):
    args = layer_args()
    with forward_ad.dual_level():
        moe.moe_forward_few(*args, 2)
        args[which] = forward_ad.make_dual(args[which], torch.ones_like(args[which]))
        with pytest.raises(RuntimeError, match="forward only"):
            moe.moe_forward_few(*args, 2)
    assert len(few_launched) == 1


@pytest.mark.parametrize("tokens", [4, 80])
def test_the_example_block_is_inference(monkeypatch, tokens):
    """Its result would otherwise have the gradient of everything but the experts."""
    monkeypatch.setattr(expert_block.norm, "layer_norm", lambda x, w, b: x * w + b)
    monkeypatch.setattr(expert_block.lora, "lora_linear", lambda x, w, a, b, adapter, scale: x @ w)
    monkeypatch.setattr(expert_block, "grouped_mm", lambda a, b: a @ b)
    for name in ("moe_forward", "moe_forward_few"):
        monkeypatch.setattr(expert_block.moe, name, lambda n, *rest: n.detach().clone())
    block = expert_block.random_block(16, 4, 2, 64, 3, 4, dtype=torch.float32, device="cpu")
    block.lora_a.requires_grad_()
    x, adapter = torch.randn(tokens, 16, requires_grad=True), torch.zeros(tokens, dtype=torch.int32)
    assert not block(x, adapter).requires_grad
    assert block.project(x, adapter).requires_grad


@pytest.fixture
def layer_stages(monkeypatch):
    """moe_forward's launches."""
    routing = moe.Routing(*(torch.zeros(8, dtype=torch.int32) for _ in range(5)))
    monkeypatch.setattr(moe, "moe_route", lambda logits, k, renormalize: routing)
    monkeypatch.setattr(moe, "_gate_up_now", lambda x, rows, w, offs: torch.zeros(8, 32, dtype=x.dtype))
    monkeypatch.setattr(moe, "grouped_mm_2d3d", lambda a, b, offs, out: None)
    monkeypatch.setattr(moe, "moe_combine", lambda y, r, tokens, k: torch.ones(tokens, y.size(1), dtype=y.dtype))


@pytest.mark.parametrize("which", range(4))
def test_the_layer_of_many_launches_raises_in_the_backward_pass(layer_stages, which):
    """It has always taken operands that require a gradient: it still does, but a gradient through it is an error."""
    args = layer_args()
    want = moe.moe_forward(*args, 2)
    assert not want.requires_grad
    args[which].requires_grad_()
    got = moe.moe_forward(*args, 2)
    assert torch.equal(got.detach(), want)
    with pytest.raises(RuntimeError, match="no gradient"):
        (args[0].float() + got.float()).sum().backward()
    with torch.no_grad():
        assert not moe.moe_forward(*args, 2).requires_grad
    with forward_ad.dual_level():
        args[which] = forward_ad.make_dual(args[which].detach(), torch.ones_like(args[which]))
        with pytest.raises(RuntimeError, match="forward-mode"):
            moe.moe_forward(*args, 2)


# ------------------------------------------------------------------ the grouped product
@pytest.mark.parametrize("through", ["sum", "cubes"])
def test_the_grouped_product_has_no_second_derivative(monkeypatch, through):
    monkeypatch.setattr(api, "validate_inputs", lambda a, b, *rest: api.Checked(False, False, a.dtype))
    monkeypatch.setattr(api._k, "grouped_mm_3d3d", lambda a, b, out: out.copy_((a.detach() @ b.detach())))
    gen = torch.Generator().manual_seed(0)
    for which in range(2):
        ab = [torch.randn(2, 3, 4, generator=gen), torch.randn(2, 4, 5, generator=gen)]
        ab[which].requires_grad_()
        y = api.grouped_mm(*ab)
        value = y.sum() if through == "sum" else (y ** 3).sum()
        first, = torch.autograd.grad(value, ab[which], retain_graph=True)
        grad, = torch.autograd.grad(value, ab[which], create_graph=True)
        assert torch.equal(first, grad.detach())
        with pytest.raises(RuntimeError, match="no second derivative"):
            (value + grad.square().sum()).backward()
