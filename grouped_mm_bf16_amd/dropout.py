"""Dropout beside a residual stream, from a counter-based generator: the mask is never stored, the backward pass makes it again.

The random bits are a function of the seed and offset in ``rng``, of ``site`` and of an element's place alone, so results are the same every time and
for every stride and type.  One launch in each direction; torch custom ops (``grouped_mm_bf16_amd::dropout``, ``dropout_backward``), which calls
dispatch to while a model around them is being traced or compiled.  The reference has no counterpart.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _lib, derivatives, kernels
from .kernels import _dtype_code, _guard, _require_gpu

STEPS = 65536      # of a probability


def _rows(x: torch.Tensor) -> torch.Tensor:
    """x as a matrix of rows whose elements are contiguous; copied only where its strides allow no such view."""
    if x.dim() != 2:
        x = x.reshape(-1, x.size(-1)) if x.numel() and x.dim() else x.reshape(1, x.numel())
    if x.is_contiguous():
        return x
    (rows, width), (step, between) = x.shape, x.stride()
    return x.contiguous() if between != 1 and width > 1 or rows > 1 and step < width else x


def _launch(x: torch.Tensor, limit: int, rng: torch.Tensor, site: int, residual: Optional[torch.Tensor], used: Optional[torch.Tensor]) -> torch.Tensor:
    rows, width = x.shape
    device, dtype = x.device, x.dtype
    out = torch.empty(rows, width, device=device, dtype=dtype)
    with _guard(x):
        rc = _lib.load().gmm_dropout(x.data_ptr(), None if residual is None else residual.data_ptr(), out.data_ptr(), rng.data_ptr(),
                                     None if used is None else used.data_ptr(), rows, width, x.stride(0),
                                     0 if residual is None else residual.stride(0), width, limit, site, _dtype_code(dtype),
                                     kernels.current_stream(device))
    _lib.check(rc, "dropout")
    return out


def _forward_now(x: torch.Tensor, limit: int, rng: torch.Tensor, site: int, residual: Optional[torch.Tensor]) -> Tuple[torch.Tensor, torch.Tensor]:
    """The result, and what rng held: the caller may count it on before the backward pass."""
    used = torch.empty_like(rng)
    return _launch(x, limit, rng, site, residual, used), used


_forward_op = torch.library.custom_op("grouped_mm_bf16_amd::dropout", mutates_args=())(_forward_now)


@_forward_op.register_fake
def _forward_fake(x, limit, rng, site, residual):
    return x.new_empty(x.shape), torch.empty_like(rng)


def _backward_now(grad: torch.Tensor, limit: int, used: torch.Tensor, site: int) -> torch.Tensor:
    return _launch(grad, limit, used, site, None, None)


_backward_op = torch.library.custom_op("grouped_mm_bf16_amd::dropout_backward", mutates_args=())(_backward_now)


@_backward_op.register_fake
def _backward_fake(grad, limit, used, site):
    return grad.new_empty(grad.shape)


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, rng, limit, site):
        impl = _forward_op if torch.compiler.is_compiling() else _forward_now
        out, used = impl(_rows(x), limit, rng, site, None if residual is None else _rows(residual))
        ctx.save_for_backward(used)
        ctx.limit, ctx.site, ctx.shape = limit, site, x.shape
        return out if x.dim() == 2 else out.reshape(x.shape)

    @staticmethod
    def backward(ctx, grad):
        used, = ctx.saved_tensors
        need_x, need_residual = ctx.needs_input_grad[:2]
        dx = None
        if need_x:
            dx = (_backward_op if torch.compiler.is_compiling() else _backward_now)(_rows(grad), ctx.limit, used, ctx.site)
            dx = dx if len(ctx.shape) == 2 else dx.reshape(ctx.shape)
        return *derivatives.gradients("dropout", dx, grad if need_residual else None), None, None, None


def dropout(x: torch.Tensor, p: float, rng: torch.Tensor, residual: Optional[torch.Tensor] = None, site: int = 0) -> torch.Tensor:
    """``residual + x * kept / (1 - p)``, each element kept with probability 1 - p, with the gradients of x and residual.

    x [...], bf16, fp16 or fp32; residual of its shape and type, or None.  p in [0, 1], a multiple of 2^-16 (rounded to one, which 1 - p follows);
    a dropped element counts as zero whatever it is.  rng int64 [2] on x's device: seed and offset.  It is read on the device: count the offset on
    (``rng[1] += 1``) after each step, also one that is replayed from a captured graph.  site in [0, 65536) tells calls apart that share rng.
    float32 arithmetic, one rounding.  Kept for the backward pass: the two numbers that rng held.
    """
    _dtype_code(x.dtype)
    limit = round(float(p) * STEPS) if 0.0 <= p <= 1.0 else -1
    if limit < 0:
        raise RuntimeError(f"dropout: p has to be in [0, 1], got {p}")
    if not 0 <= site < 65536:
        raise RuntimeError(f"dropout: site has to be in [0, 65536), got {site}")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype):
        raise RuntimeError(f"dropout: residual has to be {tuple(x.shape)} {x.dtype}, got {tuple(residual.shape)} {residual.dtype}")
    if rng.dtype != torch.int64 or rng.dim() != 1 or rng.numel() != 2 or not rng.is_contiguous():
        raise RuntimeError("dropout: rng has to be a contiguous int64 tensor of two elements, seed and offset")
    _require_gpu(x)
    if rng.device != x.device or residual is not None and residual.device != x.device:
        raise RuntimeError(f"dropout: rng and residual have to be on {x.device}")
    if ((x.requires_grad or residual is not None and residual.requires_grad) and torch.is_grad_enabled()
            or derivatives.forward_mode()):      # with a tangent it raises: there is no forward-mode derivative
        return _Dropout.apply(x, residual, rng, limit, site)
    rows, other = _rows(x), None if residual is None else _rows(residual)
    out = _forward_op(rows, limit, rng, site, other)[0] if torch.compiler.is_compiling() else _launch(rows, limit, rng, site, other, None)
    return out if x.dim() == 2 else out.reshape(x.shape)
