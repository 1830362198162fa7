"""One pre-norm block with experts, as a server or a tuner of adapters runs it through this package:

    h = x + lora_linear(layer_norm(x), projection, adapters of the tokens' requests)
    y = h + experts(layer_norm(h))

``train`` is the same with dropout beside the residual stream and the gradients of all its weights, ``eight_bit`` the same for inference with 8-bit
weights.  ``python -m grouped_mm_bf16_amd.expert_block`` decodes a few tokens and a prompt through the block and its 8-bit form, tunes its adapters and
trains it for some steps and prints the times.  The reference has no such program.
"""
from __future__ import annotations

import argparse
import time
from typing import NamedTuple

import torch

from . import dropout, grouped_mm, int8, lora, moe, moe_train, norm


def _logits(n: torch.Tensor, router: torch.Tensor) -> torch.Tensor:
    return grouped_mm(n.unsqueeze(0), router.unsqueeze(0)).squeeze(0)


class Int8Block(NamedTuple):
    """The block with 8-bit weights, without adapters; what it computes besides the products with them is in the type of its norms and router."""
    norm_in: tuple
    projection: int8.Columns  # [H, H]
    norm_experts: tuple
    router: torch.Tensor      # [H, E]
    w_up: int8.Columns        # [E, H, 2I]
    w_down: int8.Columns      # [E, I, H]
    top_k: int

    @torch.no_grad()
    def __call__(self, x: torch.Tensor) -> torch.Tensor:
        """x [T, H] -> [T, H]."""
        h = x + int8.linear_int8(norm.layer_norm(x, *self.norm_in), self.projection)
        n = norm.layer_norm(h, *self.norm_experts)
        return h + int8.moe_forward_int8(n, _logits(n, self.router), self.w_up, self.w_down, self.top_k)


class ExpertBlock(NamedTuple):
    norm_in: tuple            # weight, bias [H]
    projection: torch.Tensor  # [H, H]
    lora_a: torch.Tensor      # [L, H, R]
    lora_b: torch.Tensor      # [L, R, H]
    scale: torch.Tensor       # float32 [L]
    norm_experts: tuple
    router: torch.Tensor      # [H, E]
    w_up: torch.Tensor        # [E, H, 2I]
    w_down: torch.Tensor      # [E, I, H]
    top_k: int

    def project(self, x: torch.Tensor, adapter: torch.Tensor) -> torch.Tensor:
        """The block's first half, with gradients."""
        return x + lora.lora_linear(norm.layer_norm(x, *self.norm_in), self.projection, self.lora_a, self.lora_b, adapter, self.scale)

    @torch.no_grad()
    def __call__(self, x: torch.Tensor, adapter: torch.Tensor) -> torch.Tensor:
        """x [T, H], adapter int32 [T] (-1: none) -> [T, H]; inference: the experts have no gradient, so the result has none."""
        h = self.project(x, adapter)
        n = norm.layer_norm(h, *self.norm_experts)
        experts = moe.moe_forward_few if x.size(0) <= moe.FEW_TOKENS else moe.moe_forward
        return h + experts(n, _logits(n, self.router), self.w_up, self.w_down, self.top_k)

    def train(self, x: torch.Tensor, adapter: torch.Tensor, p: float, rng: torch.Tensor, site: int = 0) -> torch.Tensor:
        """The block with dropout of probability p in front of both sums, with gradients of x and of every weight.  rng as ``dropout`` takes it, the
        caller counts it on; two sites of it are used, ``site`` and the next."""
        low = lora.lora_linear(norm.layer_norm(x, *self.norm_in), self.projection, self.lora_a, self.lora_b, adapter, self.scale)
        h = dropout.dropout(low, p, rng, x, site)
        n = norm.layer_norm(h, *self.norm_experts)
        experts = moe_train.moe_train(n, _logits(n, self.router), self.w_up, self.w_down, self.top_k)
        return dropout.dropout(experts, p, rng, h, site + 1)

    @torch.no_grad()
    def eight_bit(self, adapter: int = -1) -> Int8Block:
        """The block for inference with weights rounded to 8 bits, an adapter's product added to the projection first (-1: none)."""
        projection = self.projection.float()
        if adapter >= 0:
            low = grouped_mm(self.lora_a[adapter, None].float(), self.lora_b[adapter, None].float())
            projection = projection + self.scale[adapter] * low[0]
        return Int8Block(self.norm_in, int8.quantize_columns(projection), self.norm_experts, self.router, int8.quantize_columns(self.w_up),
                         int8.quantize_columns(self.w_down), self.top_k)

    def weights(self) -> list:
        """Every tensor that ``train`` has a gradient of."""
        return [*self.norm_in, self.projection, self.lora_a, self.lora_b, *self.norm_experts, self.router, self.w_up, self.w_down]

    def with_weights(self, weights) -> ExpertBlock:
        """The block with other tensors for those, in their order."""
        w = list(weights)
        return self._replace(norm_in=tuple(w[:2]), projection=w[2], lora_a=w[3], lora_b=w[4], norm_experts=tuple(w[5:7]), router=w[7], w_up=w[8],
                             w_down=w[9])


def random_block(hidden: int = 2048, experts: int = 128, top_k: int = 8, inner: int = 768, adapters: int = 16, rank: int = 16,
                 dtype: torch.dtype = torch.bfloat16, device: str = "cuda", seed: int = 0) -> ExpertBlock:
    gen = torch.Generator(device=device).manual_seed(seed)
    rnd = lambda scale, *shape: torch.randn(*shape, device=device, dtype=dtype, generator=gen).mul_(scale)
    pair = lambda: (rnd(0.1, hidden).add_(1.0), rnd(0.1, hidden))
    return ExpertBlock(pair(), rnd(hidden ** -0.5, hidden, hidden), rnd(hidden ** -0.5, adapters, hidden, rank),
                       torch.zeros(adapters, rank, hidden, device=device, dtype=dtype), torch.full((adapters,), 2.0, device=device), pair(),
                       rnd(hidden ** -0.5, hidden, experts), rnd(hidden ** -0.5, experts, hidden, 2 * inner),
                       rnd(inner ** -0.5, experts, inner, hidden), top_k)


def tune(block: ExpertBlock, x: torch.Tensor, adapter: torch.Tensor, target: torch.Tensor, steps: int, rate: float) -> list:
    """Gradient steps on the adapters alone, towards ``block.project(x, adapter) == target``; the mean square error before each step.  The
    adapters of all the requests in x are tuned at once."""
    losses = []
    a, b = block.lora_a.detach().requires_grad_(), block.lora_b.detach().requires_grad_()
    for _ in range(steps):
        off = block._replace(lora_a=a, lora_b=b).project(x, adapter).float() - target.float()
        loss = off.square().mean()
        grads = torch.autograd.grad(loss, (a, b))
        losses.append(loss.detach())
        with torch.no_grad():
            for p, g in zip((a, b), grads):
                p.sub_(g.float().mul(rate).to(p.dtype))
    block.lora_a.copy_(a.detach())
    block.lora_b.copy_(b.detach())
    return [float(v) for v in losses]


def train(block: ExpertBlock, x: torch.Tensor, adapter: torch.Tensor, target: torch.Tensor, steps: int, rate: float, p: float = 0.1, seed: int = 0) -> list:
    """Gradient steps on all of the block's weights, towards ``block.train(..) == target``; the mean square error before each step."""
    losses = []
    weights = [t.detach().requires_grad_() for t in block.weights()]
    rng = torch.tensor([seed, 0], device=x.device)
    for _ in range(steps):
        off = block.with_weights(weights).train(x, adapter, p, rng).float() - target.float()
        loss = off.square().mean()
        grads = torch.autograd.grad(loss, weights)
        losses.append(loss.detach())
        rng[1] += 1
        with torch.no_grad():
            for w, g in zip(weights, grads):
                w.sub_(g.float().mul(rate).to(w.dtype))
    return [float(v) for v in losses]


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--hidden", type=int, default=2048)
    ap.add_argument("--experts", type=int, default=128)
    ap.add_argument("--active-experts-per-token", type=int, default=8)
    ap.add_argument("--inner", type=int, default=768)
    ap.add_argument("--adapters", type=int, default=16)
    ap.add_argument("--rank", type=int, default=16)
    ap.add_argument("--sequences", type=int, default=32, help="sequences of the decoding step, each with an adapter of its own choice")
    ap.add_argument("--prompt", type=int, default=2048, help="tokens of the prompt and of a tuning step")
    ap.add_argument("--steps", type=int, default=20)
    args = ap.parse_args()
    block = random_block(args.hidden, args.experts, args.active_experts_per_token, args.inner, args.adapters, args.rank)
    gen = torch.Generator(device="cuda").manual_seed(1)

    def batch(tokens: int, requests: int):
        x = torch.randn(tokens, args.hidden, device="cuda", dtype=torch.bfloat16, generator=gen)
        which = torch.randint(-1, args.adapters, (requests,), device="cuda", generator=gen)
        return x, which.repeat_interleave(-(-tokens // requests))[:tokens].to(torch.int32)

    def timed(run) -> float:
        for _ in range(5):
            run()
        torch.cuda.synchronize()
        start = time.perf_counter()
        for _ in range(args.steps):
            run()
        torch.cuda.synchronize()
        return (time.perf_counter() - start) / args.steps * 1e6

    eight = block.eight_bit()
    for what, tokens, requests in (("decoding", args.sequences, args.sequences), ("prompt", args.prompt, 4)):
        x, adapter = batch(tokens, requests)
        print(f"{what}: {tokens} tokens {timed(lambda: block(x, adapter)):.1f} us, with 8-bit weights {timed(lambda: eight(x)):.1f} us")
    x, adapter = batch(args.prompt, 4)
    target = block.project(x, adapter) + 0.1 * torch.randn(args.prompt, args.hidden, device="cuda", dtype=torch.bfloat16, generator=gen)
    tune(block, x, adapter, target, 2, 0.0)
    torch.cuda.synchronize()
    start = time.perf_counter()
    losses = tune(block, x, adapter, target, args.steps, args.hidden / 16)
    print(f"tuning: {args.prompt} tokens {(time.perf_counter() - start) / args.steps * 1e6:.1f} us a step, error {losses[0]:.5f} -> {losses[-1]:.5f}")
    train(block, x, adapter, target, 2, 0.0)
    torch.cuda.synchronize()
    start = time.perf_counter()
    losses = train(block, x, adapter, target, args.steps, 1.0)
    print(f"training: {args.prompt} tokens {(time.perf_counter() - start) / args.steps * 1e6:.1f} us a step, error {losses[0]:.5f} -> {losses[-1]:.5f}")


if __name__ == "__main__":
    main()
