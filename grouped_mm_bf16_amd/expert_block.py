"""One pre-norm block with experts, as a server or a tuner of adapters runs it through this package:

    h = x + lora_linear(layer_norm(x), projection, adapters of the tokens' requests)
    y = h + experts(layer_norm(h))

``python -m grouped_mm_bf16_amd.expert_block`` decodes a few tokens and a prompt through such a block, tunes its adapters for some steps
and prints the times.  The reference has no such program.
"""
from __future__ import annotations

import argparse
import time
from typing import NamedTuple

import torch

from . import grouped_mm, lora, moe, norm


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
        logits = grouped_mm(n.unsqueeze(0), self.router.unsqueeze(0)).squeeze(0)
        experts = moe.moe_forward_few if x.size(0) <= moe.FEW_TOKENS else moe.moe_forward
        return h + experts(n, logits, self.w_up, self.w_down, self.top_k)


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

    for what, tokens, requests in (("decoding", args.sequences, args.sequences), ("prompt", args.prompt, 4)):
        x, adapter = batch(tokens, requests)
        for _ in range(5):
            block(x, adapter)
        torch.cuda.synchronize()
        start = time.perf_counter()
        for _ in range(args.steps):
            block(x, adapter)
        torch.cuda.synchronize()
        print(f"{what}: {tokens} tokens {(time.perf_counter() - start) / args.steps * 1e6:.1f} us")
    x, adapter = batch(args.prompt, 4)
    target = block.project(x, adapter) + 0.1 * torch.randn(args.prompt, args.hidden, device="cuda", dtype=torch.bfloat16, generator=gen)
    tune(block, x, adapter, target, 2, 0.0)
    torch.cuda.synchronize()
    start = time.perf_counter()
    losses = tune(block, x, adapter, target, args.steps, args.hidden / 16)
    print(f"tuning: {args.prompt} tokens {(time.perf_counter() - start) / args.steps * 1e6:.1f} us a step, error {losses[0]:.5f} -> {losses[-1]:.5f}")


if __name__ == "__main__":
    main()
