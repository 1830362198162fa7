"""The mixture-of-experts layer with gradients, and its steps around the grouped products:

    route -> sort_rows -> grouped_mm -> gated -> grouped_mm -> combine_rows

Each step has its derivative in kernels of its own (the products have theirs in ``grouped_mm``): tokens' rows are sorted by expert and brought
back token by token, without atomics, so results and gradients are the same every time.  No count reaches the host.  The steps are torch
custom ops (``grouped_mm_bf16_amd::sort_rows``, ``sum_rows``, ``combine_backward``, ``route_backward``, ``gated``, ``gated_backward``, and
routing's ``moe_route``), which calls dispatch to while a model around them is being traced or compiled.  The reference has no counterpart.
"""
from __future__ import annotations

from typing import List, Optional

import torch

from . import _lib, derivatives, kernels, moe
from .api import grouped_mm
from .kernels import _dtype_code, _guard, _require_gpu
from .moe import ACTIVATIONS, Routing

MAX_TOP_K = 32


def _rows(x: torch.Tensor) -> torch.Tensor:
    """x with contiguous rows that do not overlap; copied only where they do not lie so."""
    if x.is_contiguous():
        return x
    (rows, width), (step, between) = x.shape, x.stride()
    if between != 1 and width > 1 or rows > 1 and step < width:
        return x.contiguous()
    return x


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


# ------------------------------------------------------------------ routing
def _route_backward_now(dweight: torch.Tensor, slot_expert: torch.Tensor, slot_weight: torch.Tensor, logits: Optional[torch.Tensor],
                        tokens: int, experts: int, top_k: int, dtype: torch.dtype) -> torch.Tensor:
    out = torch.empty(tokens, experts, device=dweight.device, dtype=dtype)
    with _guard(dweight):
        rc = _lib.load().gmm_moe_route_backward(dweight.data_ptr(), slot_expert.data_ptr(), slot_weight.data_ptr(), _ptr(logits), out.data_ptr(),
                                                tokens, experts, top_k, logits.stride(0) if logits is not None else experts, _dtype_code(dtype),
                                                kernels.current_stream(dweight.device))
    _lib.check(rc, "route backward")
    return out


_route_backward_op = torch.library.custom_op("grouped_mm_bf16_amd::route_backward", mutates_args=())(_route_backward_now)


@_route_backward_op.register_fake
def _route_backward_fake(dweight, slot_expert, slot_weight, logits, tokens, experts, top_k, dtype):
    return dweight.new_empty(tokens, experts, dtype=dtype)


class _Route(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, top_k, renormalize):
        offs, slot_expert, slot_weight, row_token, token_rows = moe.moe_route(logits, top_k, renormalize)
        ctx.mark_non_differentiable(offs, slot_expert, row_token, token_rows)
        ctx.save_for_backward(slot_expert, slot_weight, None if renormalize else logits)
        ctx.shape, ctx.dtype, ctx.top_k = logits.shape, logits.dtype, top_k
        return offs, slot_expert, slot_weight, row_token, token_rows

    @staticmethod
    def backward(ctx, _offs, _expert, grad, _token, _rows_of):
        slot_expert, slot_weight, logits = ctx.saved_tensors
        impl = _route_backward_op if torch.compiler.is_compiling() else _route_backward_now
        out = impl(grad.contiguous(), slot_expert, slot_weight, logits, *ctx.shape, ctx.top_k, ctx.dtype)
        return *derivatives.gradients("route", out), None, None


def route(router_logits: torch.Tensor, top_k: int, renormalize: bool = True) -> Routing:
    """:func:`moe.moe_route`, whose weights (``slot_weight``) have a gradient: that of the softmax over the chosen logits (``renormalize``) or
    over all.  The choice itself is a constant; the logits of experts that were not chosen get zeros, or their share of the whole softmax."""
    if router_logits.requires_grad and torch.is_grad_enabled() or derivatives.forward_mode():     # with a tangent it raises
        return Routing(*_Route.apply(router_logits, top_k, bool(renormalize)))
    return moe.moe_route(router_logits, top_k, renormalize)


# ------------------------------------------------------------------ rows sorted by expert, and back
def _check_rows(what: str, x: torch.Tensor, routing: Routing, slots: int, weights: bool) -> None:
    _dtype_code(x.dtype)
    if x.dim() != 2:
        raise RuntimeError(f"{what} takes a 2D tensor, got {x.dim()}D")
    _require_gpu(x)
    _check_routing(what, "token_rows", routing.token_rows, torch.int32, x.device, slots)
    if weights:
        _check_routing(what, "slot_weight", routing.slot_weight, torch.float32, x.device, slots)


def _check_routing(what: str, name: str, t: torch.Tensor, dtype: torch.dtype, device: torch.device, slots: int) -> None:
    if t.dtype != dtype or t.dim() != 1 or not t.is_contiguous() or t.device != device:
        raise RuntimeError(f"{what}: routing.{name} has to be a contiguous 1D {dtype} tensor on {device}, got {t.dim()}D {t.dtype} on {t.device}")
    if t.numel() != slots:
        raise RuntimeError(f"{what}: routing.{name} has to have tokens * top_k = {slots} elements, got {t.numel()}")


def _sort_now(x: torch.Tensor, token_rows: torch.Tensor) -> torch.Tensor:
    (tokens, width), slots = x.shape, token_rows.numel()
    out = torch.empty(slots, width, device=x.device, dtype=x.dtype)
    if slots:
        with _guard(x):
            rc = _lib.load().gmm_moe_sort_rows(x.data_ptr(), token_rows.data_ptr(), out.data_ptr(), tokens, slots // tokens, width, slots,
                                               x.stride(0), width, _dtype_code(x.dtype), kernels.current_stream(x.device))
        _lib.check(rc, "sort_rows")
    return out


_sort_op = torch.library.custom_op("grouped_mm_bf16_amd::sort_rows", mutates_args=())(_sort_now)


@_sort_op.register_fake
def _sort_fake(x, token_rows):
    return x.new_empty(token_rows.numel(), x.size(1))


def _sum_now(y: torch.Tensor, token_rows: torch.Tensor, slot_weight: Optional[torch.Tensor], tokens: int, top_k: int) -> torch.Tensor:
    out = torch.empty(tokens, y.size(1), device=y.device, dtype=y.dtype)
    with _guard(y):
        rc = _lib.load().gmm_moe_sum_rows(y.data_ptr(), token_rows.data_ptr(), _ptr(slot_weight), out.data_ptr(), tokens, top_k, y.size(1),
                                          y.size(0), y.stride(0), y.size(1), _dtype_code(y.dtype), kernels.current_stream(y.device))
    _lib.check(rc, "sum of rows")
    return out


_sum_op = torch.library.custom_op("grouped_mm_bf16_amd::sum_rows", mutates_args=())(_sum_now)


@_sum_op.register_fake
def _sum_fake(y, token_rows, slot_weight, tokens, top_k):
    return y.new_empty(tokens, y.size(1))


class _Sort(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, token_rows):
        ctx.save_for_backward(token_rows)
        ctx.tokens = x.size(0)
        return (_sort_op if torch.compiler.is_compiling() else _sort_now)(_rows(x), token_rows)

    @staticmethod
    def backward(ctx, grad):
        token_rows, = ctx.saved_tensors
        tokens = ctx.tokens
        out = (_sum_op if torch.compiler.is_compiling() else _sum_now)(_rows(grad), token_rows, None, tokens, token_rows.numel() // tokens if tokens else 1)
        return *derivatives.gradients("sort_rows", out), None


def sort_rows(x: torch.Tensor, routing: Routing) -> torch.Tensor:
    """``x[routing.row_token]``: each token's row once for each of its choices, sorted by expert, what ``grouped_mm`` takes with ``routing.offs``;
    its gradient adds a token's rows up in float32, in the order of its choices, and rounds once.

    x [T, H], bf16, fp16 or fp32, any H and row stride; routing of the same T tokens as :func:`route` returns it (of its tensors
    ``token_rows`` is read).  Returns [T * top_k, H].
    """
    tokens, slots = x.size(0) if x.dim() else 0, routing.token_rows.numel()
    top_k = slots // tokens if tokens else 0
    _check_rows("sort_rows", x, routing, tokens * top_k, False)
    if tokens and not 1 <= top_k <= MAX_TOP_K:
        raise RuntimeError(f"sort_rows: top_k has to be in [1, {MAX_TOP_K}], got {slots} slots for {tokens} tokens")
    if x.requires_grad and torch.is_grad_enabled() or derivatives.forward_mode():
        return _Sort.apply(x, routing.token_rows)
    return (_sort_op if torch.compiler.is_compiling() else _sort_now)(_rows(x), routing.token_rows)


def _combine_backward_now(grad: torch.Tensor, y: torch.Tensor, token_rows: torch.Tensor, slot_weight: torch.Tensor, top_k: int, need_y: bool,
                          need_weight: bool) -> List[torch.Tensor]:
    """dy and dweight (empty where not needed)."""
    tokens, width = grad.shape
    slots = token_rows.numel()
    dy = torch.empty(slots if need_y else 0, width, device=grad.device, dtype=grad.dtype)
    dw = torch.empty(slots if need_weight else 0, device=grad.device, dtype=torch.float32)
    with _guard(grad):
        rc = _lib.load().gmm_moe_combine_backward(grad.data_ptr(), y.data_ptr(), token_rows.data_ptr(), slot_weight.data_ptr(),
                                                  dy.data_ptr() if need_y else None, dw.data_ptr() if need_weight else None, tokens, top_k, width,
                                                  slots, grad.stride(0), y.stride(0), width, _dtype_code(grad.dtype),
                                                  kernels.current_stream(grad.device))
    _lib.check(rc, "combine_rows backward")
    return [dy, dw]


_combine_backward_op = torch.library.custom_op("grouped_mm_bf16_amd::combine_backward", mutates_args=())(_combine_backward_now)


@_combine_backward_op.register_fake
def _combine_backward_fake(grad, y, token_rows, slot_weight, top_k, need_y, need_weight):
    slots = token_rows.numel()
    return [grad.new_empty(slots if need_y else 0, grad.size(1)), slot_weight.new_empty(slots if need_weight else 0)]


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, slot_weight, token_rows, top_k):
        y = _rows(y)
        ctx.save_for_backward(y if ctx.needs_input_grad[1] else y.new_empty(0, y.size(1)), slot_weight, token_rows)
        ctx.top_k = top_k
        return (_sum_op if torch.compiler.is_compiling() else _sum_now)(y, token_rows, slot_weight, y.size(0) // top_k, top_k)

    @staticmethod
    def backward(ctx, grad):
        y, slot_weight, token_rows = ctx.saved_tensors
        need_y, need_weight = ctx.needs_input_grad[:2]
        impl = _combine_backward_op if torch.compiler.is_compiling() else _combine_backward_now
        dy, dw = impl(_rows(grad), y, token_rows, slot_weight, ctx.top_k, need_y, need_weight)
        return *derivatives.gradients("combine_rows", dy if need_y else None, dw if need_weight else None), None, None


def combine_rows(y: torch.Tensor, routing: Routing, top_k: int) -> torch.Tensor:
    """``sum over j < top_k of routing.slot_weight[t, j] * y[routing.token_rows[t, j]]``: the experts' rows brought back to their tokens, added up
    in float32 in the order of the choices and rounded once; with the gradients of y and of the weights.

    y [T * top_k, H], bf16, fp16 or fp32, any H and row stride; routing as :func:`route` returns it.  Returns [T, H].
    """
    if not 1 <= top_k <= MAX_TOP_K:
        raise RuntimeError(f"combine_rows: top_k has to be in [1, {MAX_TOP_K}], got {top_k}")
    slots = y.size(0) if y.dim() else 0
    _check_rows("combine_rows", y, routing, slots, True)
    if slots % top_k:
        raise RuntimeError(f"combine_rows: y has to have tokens * top_k rows, got {slots} for top_k {top_k}")
    weight, rows = routing.slot_weight, routing.token_rows
    if (y.requires_grad or weight.requires_grad) and torch.is_grad_enabled() or derivatives.forward_mode():
        return _Combine.apply(y, weight, rows, top_k)
    return (_sum_op if torch.compiler.is_compiling() else _sum_now)(_rows(y), rows, weight, slots // top_k, top_k)


# ------------------------------------------------------------------ activation
def _gated_now(h: torch.Tensor, kind: int) -> torch.Tensor:
    rows, width = h.shape
    inner, device, dtype = width // 2 if kind else width, h.device, h.dtype
    out = torch.empty(rows, inner, device=device, dtype=dtype)
    with _guard(h):
        rc = _lib.load().gmm_gated(h.data_ptr(), out.data_ptr(), rows, inner, h.stride(0), inner, kind, _dtype_code(dtype),
                                   kernels.current_stream(device))
    _lib.check(rc, "gated")
    return out


_gated_op = torch.library.custom_op("grouped_mm_bf16_amd::gated", mutates_args=())(_gated_now)


@_gated_op.register_fake
def _gated_fake(h, kind):
    return h.new_empty(h.size(0), h.size(1) // (1 + kind))


def _gated_backward_now(grad: torch.Tensor, h: torch.Tensor, kind: int) -> torch.Tensor:
    rows, width = h.shape
    device, dtype = h.device, h.dtype
    out = torch.empty(rows, width, device=device, dtype=dtype)
    with _guard(h):
        rc = _lib.load().gmm_gated_backward(grad.data_ptr(), h.data_ptr(), out.data_ptr(), rows, width // 2 if kind else width, grad.stride(0),
                                            h.stride(0), width, kind, _dtype_code(dtype), kernels.current_stream(device))
    _lib.check(rc, "gated backward")
    return out


_gated_backward_op = torch.library.custom_op("grouped_mm_bf16_amd::gated_backward", mutates_args=())(_gated_backward_now)


@_gated_backward_op.register_fake
def _gated_backward_fake(grad, h, kind):
    return h.new_empty(h.shape)


class _Gated(torch.autograd.Function):
    @staticmethod
    def forward(ctx, h, kind):
        h = _rows(h)
        ctx.save_for_backward(h)
        ctx.kind = kind
        return (_gated_op if torch.compiler.is_compiling() else _gated_now)(h, kind)

    @staticmethod
    def backward(ctx, grad):
        h, = ctx.saved_tensors
        out = (_gated_backward_op if torch.compiler.is_compiling() else _gated_backward_now)(_rows(grad), h, ctx.kind)
        return *derivatives.gradients("gated", out), None


def gated(h: torch.Tensor, kind: str = "swiglu") -> torch.Tensor:
    """``silu(h)`` or, for "swiglu", ``silu(h[:, :I]) * h[:, I:]`` with I = h.size(1) // 2, with its gradient; float32 arithmetic, one rounding.

    h [R, I or 2 I], bf16, fp16 or fp32, any I and row stride.  The backward pass reads h again: nothing else is kept for it.
    """
    if kind not in ACTIVATIONS:
        raise RuntimeError(f"unknown activation {kind!r}; have {sorted(ACTIVATIONS)}")
    code = ACTIVATIONS[kind]
    _dtype_code(h.dtype)
    if h.dim() != 2:
        raise RuntimeError(f"gated takes a 2D tensor, got {h.dim()}D")
    if code and h.size(1) % 2:
        raise RuntimeError("swiglu needs an even number of columns")
    _require_gpu(h)
    if h.requires_grad and torch.is_grad_enabled() or derivatives.forward_mode():
        return _Gated.apply(h, code)
    return (_gated_op if torch.compiler.is_compiling() else _gated_now)(_rows(h), code)


# ------------------------------------------------------------------ the layer
def moe_train(x: torch.Tensor, router_logits: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor, top_k: int, activation: str = "swiglu",
              renormalize: bool = True) -> torch.Tensor:
    """:func:`moe.moe_forward` with the gradients of x, router_logits, w_up and w_down.

    x [T, H]; router_logits [T, E]; w_up [E, H, I] ("silu") or [E, H, 2 I] ("swiglu": gate columns first, then up columns); w_down [E, I, H];
    x and the weights of one type, bf16, fp16 or fp32.  Rounds as that does, after each of the products, the activation and the sum.  Kept for the
    backward pass: the sorted rows, both products' results and the activation's.
    """
    if x.dim() != 2 or router_logits.dim() != 2 or x.size(0) != router_logits.size(0):
        raise RuntimeError("x [T, H] and router_logits [T, E] must agree on T")
    if w_up.dim() != 3 or w_down.dim() != 3 or w_up.size(0) != router_logits.size(1) or w_down.size(0) != w_up.size(0):
        raise RuntimeError("w_up [E, H, I or 2I] and w_down [E, I, H] must agree with router_logits on E")
    if activation not in ACTIVATIONS:
        raise RuntimeError(f"unknown activation {activation!r}; have {sorted(ACTIVATIONS)}")
    inner = w_up.size(2) // 2 if ACTIVATIONS[activation] else w_up.size(2)
    if w_up.size(1) != x.size(1) or w_down.size(1) != inner or w_down.size(2) != x.size(1):
        raise RuntimeError("weight shapes do not chain: x [T, H], w_up [E, H, I or 2I], w_down [E, I, H]")
    routing = route(router_logits, top_k, renormalize)
    h = grouped_mm(sort_rows(x, routing), w_up, offs=routing.offs)
    y = grouped_mm(gated(h, activation), w_down, offs=routing.offs)
    return combine_rows(y, routing, top_k)
