"""Where torch would differentiate what has no derivative here, an error and never a wrong value: the kernels take raw pointers, so torch
would treat their results as constants without a word."""
from __future__ import annotations

import torch
from torch.autograd import forward_ad


class _NoDerivative(torch.autograd.Function):
    @staticmethod
    def forward(ctx, what, _anchor, *results):
        ctx.what = what
        return results

    @staticmethod
    def backward(ctx, *_grads):
        raise RuntimeError(ctx.what)


def without_derivative(what: str, *results):
    """The results, each of them such that a backward pass that reaches it raises `what`.  (The anchor makes them require a gradient whatever
    they were computed from.)"""
    return _NoDerivative.apply(what, torch.zeros((), requires_grad=True), *results)


def gradients(name: str, *grads):
    """What a backward function returns.  Under ``create_graph=True`` a further differentiation of the gradients raises."""
    if torch.is_grad_enabled() and not torch.compiler.is_compiling():
        there = iter(without_derivative(f"{name} has no second derivative", *(g for g in grads if g is not None)))
        return tuple(None if g is None else next(there) for g in grads)
    return grads


def forward_mode() -> bool:
    """Whether a tensor may have a tangent (``forward_ad.unpack_dual`` costs 0.3 us a tensor, this 0.06)."""
    return forward_ad._current_level >= 0


def tangent(*tensors) -> bool:
    """Whether one of the tensors has a tangent."""
    return forward_mode() and any(forward_ad.unpack_dual(t).tangent is not None for t in tensors)
