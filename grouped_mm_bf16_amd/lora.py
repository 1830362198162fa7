"""A projection that all tokens share beside the low-rank adapters of many requests, and the adapters' gradients.

    y[t] = x[t] @ W + scale[i] * (x[t] @ A[i]) @ B[i],   i = adapter[t]

Which token has which adapter is device data that the host never sees, tokens come in any order, and a number outside the adapters means
none.  Up to ``FEW_TOKENS`` tokens (a decoding step) run in two kernels that read W and the adapters once, past the tokens; more run as W's
grouped product of one group, in float32, and two kernels for the adapters, the last of which rounds the sum.  Registered as torch custom ops (``grouped_mm_bf16_amd::lora``,
``lora_grad``), which calls dispatch to while a model around them is being traced or compiled.  The reference has no counterpart.
"""
from __future__ import annotations

import functools
from typing import List, Optional, Tuple

import torch

from . import _lib, derivatives, kernels
from .api import is_row_major
from .kernels import _dtype_code, _guard, _require_gpu

FEW_TOKENS = 64
MAX_RANK = 256
MAX_ADAPTERS = 1022
_DTYPES = (torch.bfloat16, torch.float16)


def _check(x: torch.Tensor, weight: torch.Tensor, lora_a: torch.Tensor, lora_b: torch.Tensor, adapter: torch.Tensor,
           scale: Optional[torch.Tensor]) -> None:
    if x.dim() != 2 or weight.dim() != 2 or lora_a.dim() != 3 or lora_b.dim() != 3:
        raise RuntimeError("lora_linear takes x [T, K], weight [K, N], lora_a [L, K, R] and lora_b [L, R, N]")
    dtype = x.dtype
    if dtype not in _DTYPES or not dtype == weight.dtype == lora_a.dtype == lora_b.dtype:
        raise RuntimeError("x, weight, lora_a and lora_b have to be of one type, bfloat16 or float16, got "
                           f"{x.dtype}, {weight.dtype}, {lora_a.dtype}, {lora_b.dtype}")
    (T, K), (inner, N), (L, Ka, R) = x.shape, weight.shape, lora_a.shape
    if K != inner or Ka != K or lora_b.shape != (L, R, N):
        raise RuntimeError("shapes do not chain: x [T, K], weight [K, N], lora_a [L, K, R], lora_b [L, R, N]")
    if not 1 <= R <= MAX_RANK:
        raise RuntimeError(f"the adapters' rank must be in [1, {MAX_RANK}], got {R}")
    if L > MAX_ADAPTERS:
        raise RuntimeError(f"Can't process more than {MAX_ADAPTERS} adapters")
    if adapter.dtype != torch.int32 or adapter.shape != (T,) or not adapter.is_contiguous():
        raise RuntimeError("adapter has to be a contiguous 1D int32 tensor with one number a row of x")
    device = x.device
    if scale is not None:
        if scale.dtype != torch.float32 or scale.shape != (L,) or not scale.is_contiguous():
            raise RuntimeError("scale has to be a contiguous 1D float32 tensor with one number an adapter")
        if scale.requires_grad:
            raise RuntimeError("scale has no gradient: it must not require one")
        if scale.device != device:
            raise RuntimeError("all operands must be on the same device")
    _require_gpu(x)
    if weight.device != device or lora_a.device != device or lora_b.device != device or adapter.device != device:
        raise RuntimeError("all operands must be on the same device")
    row, column = weight.stride()
    if not (column == 1 and row >= N or row == 1 and column >= K):
        is_row_major(weight)      # empty and single-element dimensions, or the error


def _rows(x: torch.Tensor) -> torch.Tensor:
    """x with contiguous rows that do not overlap (copied only where they do not lie so, or very far apart)."""
    if x.numel() and (x.stride(1) != 1 and x.size(1) > 1 or x.size(0) > 1 and not x.size(1) <= x.stride(0) <= 1 << 22):
        return x.contiguous()
    return x


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


@functools.lru_cache(maxsize=4096)
def _workspace_bytes(device: int, T: int, K: int, N: int, R: int) -> int:
    return _lib.load().gmm_lora_workspace_bytes(T, K, N, R)


def _rows_at_once(T: int, N: int) -> int:
    """Rows whose product with W is held in float32 at a time: 512 MiB of it, at least 2048.  Smaller parts cost rounds of tiles that are not full:
    65536 rows of 4096 -> 4096 2.07 ms in parts of 32768 rows, 2.29 in parts of 8192, 2.1 all at once."""
    return min(T, max(2048, (1 << 27) // max(N, 1) // 256 * 256))


@functools.lru_cache(maxsize=4096)
def _grad_workspace_bytes(device: int, T: int, K: int, N: int, R: int, L: int) -> int:
    return _lib.load().gmm_lora_grad_workspace_bytes(T, K, N, R, L)


def _forward_now(x: torch.Tensor, weight: torch.Tensor, lora_a: torch.Tensor, lora_b: torch.Tensor, adapter: torch.Tensor,
                 scale: Optional[torch.Tensor], save: bool) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """The result, and (with `save`) x @ lora_a of the rows that have an adapter, [T, R] float32."""
    (T, K), N, dev = x.shape, weight.size(1), x.device
    L, _, R = lora_a.shape
    if save and _grad_workspace_bytes(dev.index, T, K, N, R, L) < 0:
        raise RuntimeError(f"lora_linear: too many rows for gradients of adapters of rank {R}, or too large ones: got {T} rows, {K} to {N}")
    out = torch.empty(T, N, device=dev, dtype=x.dtype)
    low = torch.empty(T, R, device=dev, dtype=torch.float32) if save else None
    lib = _lib.load()
    with _guard(x):
        stream, code = kernels.current_stream(dev), _dtype_code(x.dtype)
        rc = _lib.ERR_UNSUPPORTED
        if T <= FEW_TOKENS:
            nbytes = _workspace_bytes(dev.index, T, K, N, R)
            ws = torch.empty(nbytes, device=dev, dtype=torch.uint8)
            rc = lib.gmm_lora_linear(x.data_ptr(), weight.data_ptr(), lora_a.data_ptr(), lora_b.data_ptr(), adapter.data_ptr(), _ptr(scale),
                                     out.data_ptr(), _ptr(low), T, K, N, R, L, x.stride(0), *weight.stride(), *lora_a.stride(),
                                     *lora_b.stride(), N, code, ws.data_ptr(), nbytes, stream)
        if rc == _lib.ERR_UNSUPPORTED:
            most = _rows_at_once(T, N)
            nbytes = max(_workspace_bytes(dev.index, rows, K, N, R) for rows in (most, (T - 1) % most + 1))     # the last part's may be more
            ws = torch.empty(nbytes, device=dev, dtype=torch.uint8)
            base = torch.empty(most, N, device=dev, dtype=torch.float32)
            for first in range(0, T, most):
                rows = min(most, T - first)
                part, product, here = (x, base, out) if rows == T else (x[first:first + rows], base[:rows], out[first:first + rows])
                if K == 0:
                    product.zero_()
                elif N:
                    kernels._launch_now(kernels.V_3D3D, part.unsqueeze(0), weight.unsqueeze(0), None, product.unsqueeze(0))
                rc = lib.gmm_lora_sum(part.data_ptr(), lora_a.data_ptr(), lora_b.data_ptr(), adapter.data_ptr() + 4 * first, _ptr(scale),
                                      product.data_ptr(), here.data_ptr(), low.data_ptr() + 4 * R * first if save else None, rows, K, N, R, L,
                                      part.stride(0), *lora_a.stride(), *lora_b.stride(), N, code, ws.data_ptr(), nbytes, stream)
                if rc:
                    break
    _lib.check(rc, "lora_linear")
    return out, low


def _forward_functional(x: torch.Tensor, weight: torch.Tensor, lora_a: torch.Tensor, lora_b: torch.Tensor, adapter: torch.Tensor,
                        scale: Optional[torch.Tensor], save: bool) -> Tuple[torch.Tensor, torch.Tensor]:
    out, low = _forward_now(x, weight, lora_a, lora_b, adapter, scale, save)
    return out, low if save else x.new_empty(0, lora_a.size(2), dtype=torch.float32)


_forward_op = torch.library.custom_op("grouped_mm_bf16_amd::lora", mutates_args=())(_forward_functional)


@_forward_op.register_fake
def _forward_fake(x, weight, lora_a, lora_b, adapter, scale, save):
    return x.new_empty(x.size(0), weight.size(1)), x.new_empty(x.size(0) if save else 0, lora_a.size(2), dtype=torch.float32)


def _grad_now(x: torch.Tensor, dy: torch.Tensor, low: torch.Tensor, u: torch.Tensor, adapter: torch.Tensor, scale: Optional[torch.Tensor],
              lora_a: torch.Tensor, lora_b: torch.Tensor, need_a: bool, need_b: bool) -> List[torch.Tensor]:
    """The gradients of lora_a and lora_b, laid out as those are (empty where not needed).  u is computed here if it is empty."""
    (T, K), N = x.shape, dy.size(1)
    L, _, R = lora_a.shape
    da = torch.empty_like(lora_a) if need_a else x.new_empty(0)
    db = torch.empty_like(lora_b) if need_b else x.new_empty(0)
    lib = _lib.load()
    with _guard(x):
        stream, code = kernels.current_stream(x.device), _dtype_code(x.dtype)
        if need_a and not u.numel() and T:
            u = torch.empty(T, R, device=x.device, dtype=torch.float32)
            nbytes = _workspace_bytes(x.device.index, T, N, K, R)
            ws = torch.empty(nbytes, device=x.device, dtype=torch.uint8)
            sl, sr, sn = lora_b.stride()
            rc = lib.gmm_lora_add(dy.data_ptr(), lora_b.data_ptr(), None, adapter.data_ptr(), None, None, u.data_ptr(), T, N, 0, R, L,
                                  dy.stride(0), sl, sn, sr, 0, 0, 0, 0, code, ws.data_ptr(), nbytes, stream)
            _lib.check(rc, "lora_linear backward")
        nbytes = _grad_workspace_bytes(x.device.index, T, K, N, R, L)
        if nbytes < 0:
            raise RuntimeError("lora_linear backward: sizes out of range")
        ws = torch.empty(nbytes, device=x.device, dtype=torch.uint8)
        rc = lib.gmm_lora_grad(x.data_ptr(), dy.data_ptr(), low.data_ptr(), u.data_ptr(), adapter.data_ptr(), _ptr(scale),
                               da.data_ptr() if need_a else None, db.data_ptr() if need_b else None, T, K, N, R, L, x.stride(0),
                               dy.stride(0), *(da.stride() if need_a else (0, 0, 0)), *(db.stride() if need_b else (0, 0, 0)), code,
                               ws.data_ptr(), nbytes, stream)
    _lib.check(rc, "lora_linear backward")
    return [da, db]


_grad_op = torch.library.custom_op("grouped_mm_bf16_amd::lora_grad", mutates_args=())(_grad_now)


@_grad_op.register_fake
def _grad_fake(x, dy, low, u, adapter, scale, lora_a, lora_b, need_a, need_b):
    return [torch.empty_like(lora_a) if need_a else x.new_empty(0), torch.empty_like(lora_b) if need_b else x.new_empty(0)]


class _Lora(torch.autograd.Function):
    """Backward = the forward with W, A and B turned (dx = dy W^T + scale (dy B^T) A^T), which also gives dy B^T, and the gradients
    of A and B from the two rank-sized products."""

    @staticmethod
    def forward(ctx, x, weight, lora_a, lora_b, adapter, scale):
        x = _rows(x)
        impl = _forward_op if torch.compiler.is_compiling() else _forward_now
        out, low = impl(x, weight, lora_a, lora_b, adapter, scale, any(ctx.needs_input_grad[2:4]))
        ctx.save_for_backward(x, weight, lora_a, lora_b, adapter, scale, low)
        return out

    @staticmethod
    def backward(ctx, grad):
        x, weight, lora_a, lora_b, adapter, scale, low = ctx.saved_tensors
        need_x, need_w, need_a, need_b = ctx.needs_input_grad[:4]
        dy = _rows(grad)
        compiling = torch.compiler.is_compiling()
        dx = dw = da = db = None
        u = None
        if need_x:
            dx, u = (_forward_op if compiling else _forward_now)(dy, weight.t(), lora_b.transpose(1, 2), lora_a.transpose(1, 2), adapter, scale, need_a)
        if need_a or need_b:
            if u is None:
                u = x.new_empty(0, dtype=torch.float32)
            da, db = (_grad_op if compiling else _grad_now)(x, dy, low, u, adapter, scale, lora_a, lora_b, need_a, need_b)
        if need_w:
            dw = torch.empty(weight.shape, device=x.device, dtype=x.dtype)
            if x.size(0) == 0:
                dw.zero_()
            elif dw.numel():
                kernels.grouped_mm_3d3d(x.t().unsqueeze(0), dy.unsqueeze(0), dw.unsqueeze(0))
        return *derivatives.gradients("lora_linear", dx, dw, da if need_a else None, db if need_b else None), None, None


def lora_linear(x: torch.Tensor, weight: torch.Tensor, lora_a: torch.Tensor, lora_b: torch.Tensor, adapter: torch.Tensor,
                scale: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``x @ weight + scale[i] * (x @ lora_a[i]) @ lora_b[i]`` with each token's own adapter i, and its gradients.

    x [T, K]; weight [K, N], row- or column-major; lora_a [L, K, R], lora_b [L, R, N], any strides (views of linear layers' weights as they
    are: ``.transpose(-2, -1)``), rank R up to 256, adapters of lower rank padded with zeros; bf16 or fp16.  adapter int32 [T]: a number outside
    [0, L), such as -1, stands for none.  scale float32 [L] (None: ones) has no gradient; x, weight, lora_a and lora_b have.
    The rank-sized products and weight's product stay in float32; the result is rounded once.
    """
    _check(x, weight, lora_a, lora_b, adapter, scale)
    if ((x.requires_grad or weight.requires_grad or lora_a.requires_grad or lora_b.requires_grad) and torch.is_grad_enabled()
            or derivatives.forward_mode()):      # with a tangent it raises: there is no forward-mode derivative
        return _Lora.apply(x, weight, lora_a, lora_b, adapter, scale)
    impl = _forward_op if torch.compiler.is_compiling() else _forward_now
    return impl(_rows(x), weight, lora_a, lora_b, adapter, scale, False)[0]
