"""Layer norm: what stands before the router and the projections of a block with experts.  Forward in one kernel, backward in two
(the second adds up the sums over the rows that the weight's and the bias's gradients are); no atomics, reproducible.

The forward is registered as a torch custom op (``grouped_mm_bf16_amd::layer_norm``, the backward as ``layer_norm_backward``), which
calls dispatch to while a model around them is being traced or compiled.  The reference has no counterpart.
"""
from __future__ import annotations

from typing import List, Optional, Tuple

import torch

from . import _lib, derivatives, kernels
from .kernels import _dtype_code, _guard, _require_gpu

MAX_WIDTH = 16384


def _check(x: torch.Tensor, weight: Optional[torch.Tensor], bias: Optional[torch.Tensor]) -> torch.dtype:
    """The rules of :func:`layer_norm`; returns the type of weight and bias."""
    _require_gpu(x)
    dtype = x.dtype
    _dtype_code(dtype)
    if x.dim() < 1:
        raise RuntimeError("layer_norm takes a tensor of at least one dimension")
    width = x.size(-1)
    if width > MAX_WIDTH:
        raise RuntimeError(f"layer_norm takes rows of up to {MAX_WIDTH} elements, got {width}")
    param_dtype = None
    for t in (weight, bias):
        if t is None:
            continue
        name = "bias" if t is bias else "weight"
        if t.shape != (width,) or not t.is_contiguous():
            raise RuntimeError(f"layer_norm: {name} has to be a contiguous 1D tensor of {width} elements, got {tuple(t.shape)}")
        if t.device != x.device:
            raise RuntimeError(f"layer_norm: {name} has to be on {x.device}, got {t.device}")
        if t.dtype != dtype and t.dtype != torch.float32 or param_dtype is not None and t.dtype != param_dtype:
            raise RuntimeError(f"layer_norm: weight and bias have to be {dtype} or both float32, got {t.dtype}")
        param_dtype = t.dtype
    return param_dtype or dtype


def _rows(x: torch.Tensor) -> torch.Tensor:
    """x as a matrix of rows whose elements are contiguous; copied only where its strides allow no such view."""
    if x.dim() != 2:
        x = x.reshape(-1, x.size(-1)) if x.size(-1) else x.new_empty(0, 0)
    if x.numel() and (x.stride(1) != 1 and x.size(1) > 1 or x.size(0) > 1 and x.stride(0) < x.size(1)):
        x = x.contiguous()
    return x


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _forward_now(x: torch.Tensor, weight: Optional[torch.Tensor], bias: Optional[torch.Tensor], eps: float,
                 save: bool) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """The norm of a matrix's rows, and (with `save`) the rows' mean and rstd [2, rows]."""
    code = _dtype_code(weight.dtype if weight is not None else bias.dtype if bias is not None else x.dtype)
    rows, width = x.shape
    out = torch.empty(rows, width, device=x.device, dtype=x.dtype)
    stats = torch.empty(2, rows, device=x.device, dtype=torch.float32) if save else None
    mean = stats.data_ptr() if save else None
    with _guard(x):
        rc = _lib.load().gmm_layer_norm(x.data_ptr(), _ptr(weight), _ptr(bias), out.data_ptr(), mean, mean + 4 * rows if save else None,
                                        rows, width, x.stride(0), width, eps, _dtype_code(x.dtype), code,
                                        kernels.current_stream(x.device))
    _lib.check(rc, "layer_norm")
    return out, stats


def _forward_functional(x: torch.Tensor, weight: Optional[torch.Tensor], bias: Optional[torch.Tensor], eps: float,
                        save: bool) -> Tuple[torch.Tensor, torch.Tensor]:
    out, stats = _forward_now(x, weight, bias, eps, save)
    return out, stats if save else x.new_empty(0, dtype=torch.float32)


_forward_op = torch.library.custom_op("grouped_mm_bf16_amd::layer_norm", mutates_args=())(_forward_functional)


@_forward_op.register_fake
def _forward_fake(x, weight, bias, eps, save):
    return x.new_empty(x.shape), x.new_empty((2, x.size(0)) if save else (0,), dtype=torch.float32)


def _backward_now(dy: torch.Tensor, x: torch.Tensor, weight: Optional[torch.Tensor], stats: torch.Tensor, param_dtype: torch.dtype,
                  need_x: bool, need_weight: bool, need_bias: bool) -> List[torch.Tensor]:
    """dx, dweight, dbias (empty where not needed)."""
    rows, width = x.shape
    dev = x.device
    dx = torch.empty(rows if need_x else 0, width, device=dev, dtype=x.dtype)
    dw = torch.empty(width if need_weight else 0, device=dev, dtype=param_dtype)
    db = torch.empty(width if need_bias else 0, device=dev, dtype=param_dtype)
    lib = _lib.load()
    with _guard(x):
        nbytes = lib.gmm_layer_norm_workspace_bytes(rows, width) if need_weight or need_bias else 0
        ws = torch.empty(nbytes, device=dev, dtype=torch.uint8)
        rc = lib.gmm_layer_norm_backward(dy.data_ptr(), x.data_ptr(), _ptr(weight), stats.data_ptr(), stats.data_ptr() + 4 * rows,
                                         dx.data_ptr() if need_x else None, dw.data_ptr() if need_weight else None,
                                         db.data_ptr() if need_bias else None, rows, width, dy.stride(0), x.stride(0), width,
                                         _dtype_code(x.dtype), _dtype_code(param_dtype), ws.data_ptr(), nbytes,
                                         kernels.current_stream(dev))
    _lib.check(rc, "layer_norm backward")
    return [dx, dw, db]


_backward_op = torch.library.custom_op("grouped_mm_bf16_amd::layer_norm_backward", mutates_args=())(_backward_now)


@_backward_op.register_fake
def _backward_fake(dy, x, weight, stats, param_dtype, need_x, need_weight, need_bias):
    width = x.size(1)
    return [x.new_empty(x.size(0) if need_x else 0, width), x.new_empty(width if need_weight else 0, dtype=param_dtype),
            x.new_empty(width if need_bias else 0, dtype=param_dtype)]


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        param_dtype = _check(x, weight, bias)
        rows = _rows(x)
        save = any(ctx.needs_input_grad[:3])
        impl = _forward_op if torch.compiler.is_compiling() else _forward_now
        out, stats = impl(rows, weight, bias, float(eps), save)
        if save:
            ctx.save_for_backward(rows, weight, stats)
            ctx.param_dtype, ctx.shape = param_dtype, x.shape
        return out if x.dim() == 2 else out.reshape(x.shape)

    @staticmethod
    def backward(ctx, grad):
        x, weight, stats = ctx.saved_tensors
        dy = _rows(grad)
        impl = _backward_op if torch.compiler.is_compiling() else _backward_now
        need = ctx.needs_input_grad
        dx, dw, db = impl(dy, x, weight, stats, ctx.param_dtype, need[0], need[1], need[2])
        if need[0]:
            dx = dx if len(ctx.shape) == 2 else dx.reshape(ctx.shape)
        return *derivatives.gradients("layer_norm", dx if need[0] else None, dw if need[1] else None, db if need[2] else None), None


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5) -> torch.Tensor:
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last dimension, with its gradients.

    x [..., W], bf16, fp16 or fp32, W up to 16384; weight and bias [W] in x's type or in float32 (None: ones, zeros).  Sums in fp32, one
    rounding.  A matrix whose rows lie apart is read as it is; other tensors are copied unless they are contiguous.
    """
    if ((x.requires_grad or weight is not None and weight.requires_grad or bias is not None and bias.requires_grad) and torch.is_grad_enabled()
            or derivatives.forward_mode()):      # with a tangent it raises: there is no forward-mode derivative
        return _LayerNorm.apply(x, weight, bias, eps)
    _check(x, weight, bias)
    impl = _forward_op if torch.compiler.is_compiling() else _forward_now
    out = impl(_rows(x), weight, bias, float(eps), False)[0]
    return out if x.dim() == 2 else out.reshape(x.shape)
