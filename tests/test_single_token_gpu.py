"""Logits of one token on a real MI355X: whatever their rows' stride says, there is no second row for it to lead to."""
import pytest
import torch

from grouped_mm_bf16_amd import int8, moe, moe_train

pytestmark = pytest.mark.gpu
DEV = "cuda"


def turned(z):
    """[1, E] of strides (1, 1): a column of a contiguous [E, 1] matrix."""
    t = z.reshape(-1, 1).clone().t()
    assert t.shape == z.shape and t.stride() == (1, 1) and t.is_contiguous()
    return t


@pytest.mark.parametrize("make", [turned, lambda z: z.expand(3, -1)[:1], lambda z: z.as_strided(z.shape, (0, 1))])
@pytest.mark.parametrize("renormalize", [False, True])
@pytest.mark.parametrize("E,k", [(1, 1), (8, 2), (130, 8), (300, 32)])
def test_routing_and_its_gradient(E, k, renormalize, make):
    z = torch.randn(1, E, device=DEV, generator=torch.Generator(device=DEV).manual_seed(E))
    grad = torch.randn(k, device=DEV)
    results = []
    for logits in (z, make(z)):
        leaf = logits.detach().requires_grad_()
        r = moe_train.route(leaf, k, renormalize)
        results.append((*(t.detach() for t in r), *moe.moe_route(logits, k, renormalize), *torch.autograd.grad(r.slot_weight, leaf, grad)))
    assert all(torch.equal(p, q) for p, q in zip(*results))


@pytest.mark.parametrize("H,inner", [(135, 64), (136, 63), (136, 64)])
def test_layers(H, inner):
    gen = torch.Generator(device=DEV).manual_seed(H + inner)
    rnd = lambda *shape: torch.randn(*shape, device=DEV, generator=gen).to(torch.bfloat16)
    x, z, up, down = rnd(1, H), torch.randn(1, 6, device=DEV, generator=gen), rnd(6, H, 2 * inner), rnd(6, inner, H)
    up8, down8 = int8.quantize_columns(up), int8.quantize_columns(down)
    layers = [lambda l: int8.moe_forward_int8(x, l, up8, down8, 2), lambda l: moe_train.moe_train(x, l, up, down, 2)]
    if H % 8 == 0 and inner % 8 == 0:      # the sizes these two take
        layers += [lambda l: moe.moe_forward(x, l, up, down, 2), lambda l: moe.moe_forward_few(x, l, up, down, 2)]
    for layer in layers:
        assert torch.equal(layer(z), layer(turned(z)))
