"""Products on 8-bit integers with a scale for each token (row of the first operand) and each channel (column of the second), for serving: a linear
layer, the grouped product, and the whole mixture-of-experts layer, whose activations are rounded to 8 bits in front of both products.

    y[t, n] = a.scale[t] * b.scale[n] * sum over k of a.values[t, k] * b.values[k, n]

Weights are rounded once (:func:`quantize_columns`), activations in each call (:func:`quantize_rows`).  Sums are exact, scales are applied in
float32, the result is rounded once.  No count reaches the host.  Past a few rows weights are streamed, more go through tiles.
Registered as torch custom ops (``grouped_mm_bf16_amd::int8_quantize``, ``int8_mm``, ``int8_linear``, ``int8_layer``), which calls dispatch to while a
model around them is being traced or compiled.  Forward only.  The reference has no counterpart.
"""
from __future__ import annotations

import functools
from typing import NamedTuple, Optional, Tuple

import torch

from . import _lib, derivatives, kernels, moe, moe_train
from .kernels import _dtype_code, _guard, _require_gpu
from .moe import ACTIVATIONS

MAX_K = 131071       # sums of products of -128 .. 127 stay below 2^31
MAX_GATHERED = 1 << 31     # bytes of rows that are gathered


class Rows(NamedTuple):
    """A matrix whose rows have a scale each: row t stands for ``scale[t] * values[t]``."""
    values: torch.Tensor     # int8 [T, K]
    scale: torch.Tensor      # float32 [T]


class Columns(NamedTuple):
    """A matrix, or one for each group, whose columns have a scale each: column n stands for ``scale[n] * values[:, n]``."""
    values: torch.Tensor     # int8 [K, N] or [G, K, N], contiguous along K
    scale: torch.Tensor      # float32 [N] or [G, N]


FEW_ROWS = 64        # up to which a linear layer rounds its rows and streams the weights past them in one call
FEW_TOKENS = 256     # up to which an expert layer does, if its experts have 32 rows each or fewer (up to FEW_ROWS tokens: any number)


@functools.lru_cache(maxsize=4096)
def _linear_bytes(device: int, T: int, K: int, N: int, code: int) -> int:
    return _lib.load().gmm_int8_linear_workspace_bytes(T, K, N, code)


@functools.lru_cache(maxsize=4096)
def _layer_bytes(device: int, T: int, E: int, top_k: int, H: int, inner: int, kind: int) -> int:
    return _lib.load().gmm_int8_moe_few_workspace_bytes(T, E, top_k, H, inner, kind)


def _pitch(width: int) -> int:
    """Bytes from one row (or column) to the next: a multiple of 16."""
    return max(16, (width + 15) // 16 * 16)


def _forward_only(what: str, x: torch.Tensor, other: Optional[torch.Tensor] = None) -> None:
    if (x.requires_grad or other is not None and other.requires_grad) and torch.is_grad_enabled() or (
            derivatives.forward_mode() and derivatives.tangent(*(t for t in (x, other) if t is not None))):
        raise RuntimeError(f"{what} is forward only: call it under torch.no_grad(), or with detached operands")


# ------------------------------------------------------------------ rounding
def _quantize_now(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """values [rows, pitch], of which a row's first x.size(1) count, and scales."""
    rows, width = x.shape
    values = torch.empty(rows, _pitch(width), device=x.device, dtype=torch.int8)
    scale = torch.empty(rows, device=x.device, dtype=torch.float32)
    with _guard(x):
        rc = _lib.load().gmm_int8_quantize(x.data_ptr(), values.data_ptr(), scale.data_ptr(), rows, width, x.stride(0), values.size(1),
                                           _dtype_code(x.dtype), kernels.current_stream(x.device))
    _lib.check(rc, "quantize_rows")
    return values, scale


_quantize_op = torch.library.custom_op("grouped_mm_bf16_amd::int8_quantize", mutates_args=())(_quantize_now)


@_quantize_op.register_fake
def _quantize_fake(x):
    return x.new_empty(x.size(0), _pitch(x.size(1)), dtype=torch.int8), x.new_empty(x.size(0), dtype=torch.float32)


def _quantize(x: torch.Tensor) -> Rows:
    values, scale = (_quantize_op if torch.compiler.is_compiling() else _quantize_now)(moe_train._rows(x))
    return Rows(values[:, :x.size(1)], scale)


def quantize_rows(x: torch.Tensor) -> Rows:
    """Each row of x rounded to whole steps of a 127th of its largest magnitude (of 2^-100 at least), ties to even.

    x [T, K], bf16, fp16 or fp32, any row stride.  A row with an infinity or NaN has it as its scale, and products with it are NaN.  The values' rows
    lie at multiples of 16 bytes, as the products want them.
    """
    _dtype_code(x.dtype)
    if x.dim() != 2:
        raise RuntimeError(f"quantize_rows takes a 2D tensor, got {x.dim()}D")
    _require_gpu(x)
    _forward_only("quantize_rows", x)
    return _quantize(x)


def quantize_columns(w: torch.Tensor) -> Columns:
    """Each column of a weight matrix [K, N], or of one for each group [G, K, N], as :func:`quantize_rows` has rows: bf16, fp16 or fp32, any
    strides (a linear layer's weight as it is: ``weight.t()``).  Done once, when the weights are loaded."""
    _dtype_code(w.dtype)
    if w.dim() not in (2, 3):
        raise RuntimeError(f"quantize_columns takes a 2D or 3D tensor, got {w.dim()}D")
    _require_gpu(w)
    _forward_only("quantize_columns", w)
    turned = w.transpose(-2, -1)
    rows = _quantize(turned.reshape(turned.shape[:-1].numel(), w.size(-2)))
    return Columns(rows.values.unflatten(0, turned.shape[:-1]).transpose(-2, -1), rows.scale.reshape(turned.shape[:-1]))


# ------------------------------------------------------------------ products
def _aligned(values: torch.Tensor) -> torch.Tensor:
    """Rows [.., R, K] contiguous along K at multiples of 16 bytes; copied only where they do not lie so."""
    K = values.size(-1)
    lies = values.data_ptr() % 16 == 0
    for d in range(values.dim() - 1):
        lies = lies and (values.size(d) == 1 or values.stride(d) % 16 == 0 and values.stride(d) >= (K if d == values.dim() - 2 else 0))
    if lies and (values.stride(-1) == 1 or K == 1):
        return values
    own = torch.empty(*values.shape[:-1], _pitch(K), device=values.device, dtype=torch.int8)[..., :K]
    return own.copy_(values)


def _columns(values: torch.Tensor) -> Tuple[torch.Tensor, int, int]:
    """Columns [K, N] or [G, K, N], contiguous along K, copied only where they do not lie at multiples of 16 bytes; and the bytes from one group, one
    column to the next."""
    *lead, K, N = values.shape
    stride = values.stride()
    sg, sn = stride[0] if lead and lead[0] > 1 else 0, stride[-1] if N > 1 else _pitch(K)
    if (values.data_ptr() | sg | sn) & 15 or sn < K:
        values = _aligned(values.transpose(-2, -1)).transpose(-2, -1)
        stride = values.stride()
        sg, sn = stride[0] if lead and lead[0] > 1 else 0, stride[-1] if N > 1 else _pitch(K)
    return values, sg, sn


def _mm_now(a: torch.Tensor, a_scale: torch.Tensor, row_index: Optional[torch.Tensor], b: torch.Tensor, b_scale: torch.Tensor,
            offs: Optional[torch.Tensor], out_dtype: torch.dtype) -> torch.Tensor:
    """b [G, K, N], or without offs [K, N]."""
    G, (K, N) = 1 if offs is None else b.size(0), b.shape[-2:]
    M = a.size(0) if row_index is None else row_index.numel()
    out = torch.empty(M, N, device=a.device, dtype=out_dtype)
    if out.numel() == 0:
        return out
    if K == 0 or a.size(0) == 0:      # every row_index is outside a
        return out.zero_()
    a, (b, sg, sn) = _aligned(a), _columns(b)
    lib = _lib.load()
    with _guard(a):
        args = (a.data_ptr(), a_scale.data_ptr(), None if row_index is None else row_index.data_ptr(), b.data_ptr(), b_scale.data_ptr(), out.data_ptr(),
                None if offs is None else offs.data_ptr(), G, a.size(0), M, N, K, a.stride(0) if a.size(0) > 1 else _pitch(K), sg, sn, N,
                _dtype_code(out_dtype))
        rc = kernels.call_with_workspace(lib.gmm_int8_mm, args, a.device, kernels.current_stream(a.device))
    _lib.check(rc, "int8 product")
    return out


_mm_op = torch.library.custom_op("grouped_mm_bf16_amd::int8_mm", mutates_args=())(_mm_now)


@_mm_op.register_fake
def _mm_fake(a, a_scale, row_index, b, b_scale, offs, out_dtype):
    return a.new_empty(a.size(0) if row_index is None else row_index.numel(), b.size(-1), dtype=out_dtype)


def _mm(a: Rows, row_index: Optional[torch.Tensor], b: Columns, offs: Optional[torch.Tensor], out_dtype: torch.dtype) -> torch.Tensor:
    return (_mm_op if torch.compiler.is_compiling() else _mm_now)(a.values, a.scale, row_index, b.values, b.scale, offs, out_dtype)


def _check_columns(what: str, b: Columns, device: torch.device, dims: int) -> None:
    values, scale = b
    if values.dtype != torch.int8 or values.dim() != dims:
        raise RuntimeError(f"{what}: the columns' values have to be {dims}D int8, got {values.dim()}D {values.dtype}")
    *lead, K, N = values.shape
    if scale.dtype != torch.float32 or scale.shape != (*lead, N) or not scale.is_contiguous():
        raise RuntimeError(f"{what}: the columns' scale has to be a contiguous float32 tensor {(*lead, N)}, got {tuple(scale.shape)} {scale.dtype}")
    if K > 1 and values.stride()[-2] != 1 and values.numel():
        raise RuntimeError(f"{what}: the columns' values have to be contiguous along K, as quantize_columns lays them out; got strides {tuple(values.stride())}")
    if K > MAX_K:
        raise RuntimeError(f"{what}: K is at most {MAX_K}, got {K}")
    if values.device != device or scale.device != device:
        raise RuntimeError(f"{what}: all operands have to be on {device}")
    if scale.requires_grad or derivatives.forward_mode():
        _forward_only(what, scale)


def _check_rows(what: str, a: Rows, K: int) -> None:
    if a.values.dtype != torch.int8 or a.values.dim() != 2:
        raise RuntimeError(f"{what}: the rows' values have to be 2D int8, got {a.values.dim()}D {a.values.dtype}")
    if a.scale.dtype != torch.float32 or a.scale.shape != a.values.shape[:1] or not a.scale.is_contiguous():
        raise RuntimeError(f"{what}: the rows' scale has to be a contiguous float32 tensor ({a.values.size(0)},), got {tuple(a.scale.shape)} {a.scale.dtype}")
    if a.scale.device != a.values.device:
        raise RuntimeError(f"{what}: all operands have to be on {a.values.device}")
    _forward_only(what, a.scale)
    if a.values.size(1) != K:
        raise RuntimeError(f"{what}: contraction dimensions have to match, got {a.values.size(1)} and {K}")


def _check_groups(what: str, b: Columns, offs: torch.Tensor) -> None:
    if offs.dtype != torch.int32 or offs.dim() != 1 or not offs.is_contiguous():
        raise RuntimeError("Offsets have to be int32")
    if offs.numel() != b.values.size(0):
        raise RuntimeError("matrix batch sizes have to match")
    if offs.numel() >= 1024:
        raise RuntimeError("Can't process more than 1024 groups")
    if offs.device != b.values.device:
        raise RuntimeError(f"{what}: all operands have to be on {b.values.device}")


def int8_mm(a: Rows, b: Columns, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``(a.scale[:, None] * a.values) @ (b.values * b.scale)`` [T, N] in out_dtype (bf16, fp16 or fp32): a.values [T, K], b.values [K, N].

    Values may be any of -128 .. 127, K is at most 131071.  Operands whose rows and columns lie at multiples of 16 bytes are taken as they are, others
    copied first.
    """
    _dtype_code(out_dtype)
    _check_columns("int8_mm", b, a.values.device, 2)
    _check_rows("int8_mm", a, b.values.size(0))
    _require_gpu(a.values)
    return _mm(a, None, b, None, out_dtype)


def grouped_int8_mm(a: Rows, b: Columns, offs: torch.Tensor, out_dtype: torch.dtype = torch.bfloat16,
                    row_index: Optional[torch.Tensor] = None) -> torch.Tensor:
    """:func:`int8_mm` of jagged rows: rows offs[g - 1] .. offs[g] - 1 of the result are those of a times b's matrix g.

    a.values [M, K], b.values [G, K, N], offs int32 [G].  With row_index (int32 [M]) row m is row row_index[m] of a, which then has less than 2 GiB; a number
    outside a reads a row of zeros.  Rows past the last offset are left uninitialised, as ``grouped_mm`` leaves them.
    """
    _dtype_code(out_dtype)
    _check_columns("grouped_int8_mm", b, a.values.device, 3)
    _check_rows("grouped_int8_mm", a, b.values.size(1))
    _check_groups("grouped_int8_mm", b, offs)
    if row_index is not None and (row_index.dtype != torch.int32 or row_index.dim() != 1 or not row_index.is_contiguous()):
        raise RuntimeError("row_index has to be a contiguous 1D int32 tensor")
    if row_index is not None and row_index.device != a.values.device:
        raise RuntimeError(f"grouped_int8_mm: all operands have to be on {a.values.device}")
    _require_gpu(a.values)
    return _mm(a, row_index, b, offs, out_dtype)


def _linear_now(x: torch.Tensor, values: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    x = x if x.is_contiguous() else moe_train._rows(x)
    (T, K), N = x.shape, values.size(1)
    if 0 < T <= FEW_ROWS and N:
        b, _, sn = _columns(values)
        out = torch.empty(T, N, device=x.device, dtype=x.dtype)
        with _guard(x):
            code = _dtype_code(x.dtype)
            nbytes = _linear_bytes(x.device.index, T, K, N, code)
            ws = torch.empty(nbytes, device=x.device, dtype=torch.uint8) if nbytes > 0 else None
            rc = _lib.load().gmm_int8_linear(x.data_ptr(), b.data_ptr(), scale.data_ptr(), out.data_ptr(), T, K, N, x.stride(0), sn,
                                             N, code, None if ws is None else ws.data_ptr(), nbytes, kernels.current_stream(x.device))
        if rc != _lib.ERR_UNSUPPORTED:
            _lib.check(rc, "linear_int8")
            return out
    return _mm(_quantize(x), None, Columns(values, scale), None, x.dtype)


_linear_op = torch.library.custom_op("grouped_mm_bf16_amd::int8_linear", mutates_args=())(_linear_now)


@_linear_op.register_fake
def _linear_fake(x, values, scale):
    return x.new_empty(x.size(0), values.size(1))


def linear_int8(x: torch.Tensor, weight: Columns) -> torch.Tensor:
    """``int8_mm(quantize_rows(x), weight)`` in x's type: x [T, K], bf16, fp16 or fp32; weight of :func:`quantize_columns`, [K, N].  Forward only."""
    _dtype_code(x.dtype)
    if x.dim() != 2:
        raise RuntimeError(f"linear_int8 takes a 2D tensor, got {x.dim()}D")
    _check_columns("linear_int8", weight, x.device, 2)
    if x.size(1) != weight.values.size(0):
        raise RuntimeError(f"linear_int8: contraction dimensions have to match, got {x.size(1)} and {weight.values.size(0)}")
    _require_gpu(x)
    _forward_only("linear_int8", x)
    return (_linear_op if torch.compiler.is_compiling() else _linear_now)(x, weight.values, weight.scale)


# ------------------------------------------------------------------ the expert layer
def _gated_now(h: torch.Tensor, kind: int) -> Tuple[torch.Tensor, torch.Tensor]:
    rows, inner = h.size(0), h.size(1) // (1 + kind)
    values = torch.empty(rows, _pitch(inner), device=h.device, dtype=torch.int8)
    scale = torch.empty(rows, device=h.device, dtype=torch.float32)
    with _guard(h):
        rc = _lib.load().gmm_int8_gated(h.data_ptr(), values.data_ptr(), scale.data_ptr(), rows, inner, h.stride(0), values.size(1), kind,
                                        kernels.current_stream(h.device))
    _lib.check(rc, "int8 activation")
    return values, scale


def _activated(a: Rows, routing: moe.Routing, up: torch.Tensor, up_scale: torch.Tensor, kind: int) -> Tuple[torch.Tensor, torch.Tensor]:
    """The first product's activations in 8 bits; SwiGLU in the product's own kernel where that takes its columns."""
    b, sg, sn = _columns(up)
    (G, K, N), M = b.shape, routing.row_token.numel()
    if kind and M and K and N % 128 == 0:
        rows = _aligned(a.values)
        act = torch.empty(M, N // 2, device=rows.device, dtype=torch.float32)
        with _guard(rows):
            rc = _lib.load().gmm_int8_gate_up(rows.data_ptr(), a.scale.data_ptr(), routing.row_token.data_ptr(), b.data_ptr(), up_scale.data_ptr(),
                                              act.data_ptr(), routing.offs.data_ptr(), G, rows.size(0), M, N, K,
                                              rows.stride(0) if rows.size(0) > 1 else _pitch(K), sg, sn, N // 2, kernels.current_stream(rows.device))
        if rc != _lib.ERR_UNSUPPORTED:
            _lib.check(rc, "moe_forward_int8: first product")
            return _quantize_now(act)
        del act
    return _gated_now(_mm_now(a.values, a.scale, routing.row_token, b, up_scale, routing.offs, torch.float32), kind)


def _summed(y: torch.Tensor, routing: moe.Routing, tokens: int, top_k: int, dtype: torch.dtype) -> torch.Tensor:
    """The weighted sums of the experts' rows, which stay in fp32 until then: rounded to 16 bits they were wrong by as much again as the result's own
    rounding, and infinite in fp16 where the sum need not be."""
    out = torch.empty(tokens, y.size(1), device=y.device, dtype=dtype)
    with _guard(y):
        rc = _lib.load().gmm_moe_sum_rows_f32(y.data_ptr(), routing.token_rows.data_ptr(), routing.slot_weight.data_ptr(), out.data_ptr(), tokens, top_k,
                                              y.size(1), y.size(0), y.stride(0), y.size(1), _dtype_code(dtype), kernels.current_stream(y.device))
    _lib.check(rc, "moe_forward_int8: sum of rows")
    return out


def _layer_now(x: torch.Tensor, router_logits: torch.Tensor, up: torch.Tensor, up_scale: torch.Tensor, down: torch.Tensor, down_scale: torch.Tensor,
               top_k: int, kind: int, renormalize: bool) -> torch.Tensor:
    (T, H), (E, inner, _) = x.shape, down.shape
    if 0 < T <= FEW_TOKENS:
        rows = x if x.is_contiguous() else moe_train._rows(x)
        (b, up_g, up_n), (d, down_g, down_n) = _columns(up), _columns(down)
        logits = router_logits if T == 1 and router_logits.stride(1) == 1 else moe_train._rows(router_logits)
        with _guard(x):
            nbytes = _layer_bytes(x.device.index, T, E, top_k, H, inner, kind)
            if nbytes >= 0:
                out = torch.empty(T, H, device=x.device, dtype=x.dtype)
                ws = torch.empty(nbytes, device=x.device, dtype=torch.uint8)
                rc = _lib.load().gmm_int8_moe_few(rows.data_ptr(), logits.data_ptr(), b.data_ptr(), up_scale.data_ptr(), d.data_ptr(),
                                                  down_scale.data_ptr(), out.data_ptr(), T, E, top_k, H, inner, rows.stride(0), logits.stride(0),
                                                  up_g, up_n, down_g, down_n, H, kind, renormalize, _dtype_code(x.dtype),
                                                  _dtype_code(router_logits.dtype), ws.data_ptr(), nbytes, kernels.current_stream(x.device))
        if nbytes >= 0 and rc != _lib.ERR_UNSUPPORTED:
            _lib.check(rc, "moe_forward_int8")
            return out
    most = MAX_GATHERED // _pitch(H) - 1
    if T > most:      # tokens do not depend on one another
        parts = -(-T // most)
        return torch.cat([_layer_now(x_, z_, up, up_scale, down, down_scale, top_k, kind, renormalize)
                          for x_, z_ in zip(x.tensor_split(parts), router_logits.tensor_split(parts))])
    routing = moe.moe_route(moe_train._rows(router_logits), top_k, renormalize)
    values, scale = _activated(_quantize(x), routing, up, up_scale, kind)
    return _summed(_mm_now(values[:, :inner], scale, None, down, down_scale, routing.offs, torch.float32), routing, T, top_k, x.dtype)


_layer_op = torch.library.custom_op("grouped_mm_bf16_amd::int8_layer", mutates_args=())(_layer_now)


@_layer_op.register_fake
def _layer_fake(x, router_logits, up, up_scale, down, down_scale, top_k, kind, renormalize):
    return x.new_empty(x.shape)


def moe_forward_int8(x: torch.Tensor, router_logits: torch.Tensor, w_up: Columns, w_down: Columns, top_k: int, activation: str = "swiglu",
                     renormalize: bool = True) -> torch.Tensor:
    """:func:`moe.moe_forward` on 8-bit weights, for any number of tokens: x and the activations are rounded as :func:`quantize_rows` does, in front of
    either product.

    x [T, H], bf16 or fp16; router_logits [T, E]; w_up of :func:`quantize_columns`, [E, H, I] ("silu") or [E, H, 2 I] ("swiglu": gate columns first);
    w_down [E, I, H].  The activation takes the first product in float32, the weighted sum the second, and is rounded once.  Forward only.
    """
    if x.dim() != 2 or router_logits.dim() != 2 or x.size(0) != router_logits.size(0):
        raise RuntimeError("x [T, H] and router_logits [T, E] must agree on T")
    if x.dtype != torch.bfloat16 and x.dtype != torch.float16:
        raise RuntimeError(f"moe_forward_int8: x has to be bfloat16 or float16, got {x.dtype}")
    if activation not in ACTIVATIONS:
        raise RuntimeError(f"unknown activation {activation!r}; have {sorted(ACTIVATIONS)}")
    kind = ACTIVATIONS[activation]
    _check_columns("moe_forward_int8", w_up, x.device, 3)
    _check_columns("moe_forward_int8", w_down, x.device, 3)
    E = router_logits.size(1)
    if w_up.values.size(0) != E or w_down.values.size(0) != E:
        raise RuntimeError("w_up [E, H, I or 2I] and w_down [E, I, H] must agree with router_logits on E")
    if w_up.values.shape[1:] != (x.size(1), w_down.values.size(1) * (1 + kind)) or w_down.values.size(2) != x.size(1):
        raise RuntimeError("weight shapes do not chain: x [T, H], w_up [E, H, I or 2I], w_down [E, I, H]")
    _require_gpu(x, router_logits)
    if router_logits.device != x.device:
        raise RuntimeError(f"moe_forward_int8: all operands have to be on {x.device}")
    _forward_only("moe_forward_int8", x, router_logits)
    if not 1 <= top_k <= min(E, 32):
        raise RuntimeError(f"top_k must be in [1, min(experts, 32)], got {top_k} for {E} experts")
    if E > 1023:
        raise RuntimeError("Can't process more than 1024 groups")
    _dtype_code(router_logits.dtype)
    return (_layer_op if torch.compiler.is_compiling() else _layer_now)(x, router_logits, *w_up, *w_down, top_k, kind, bool(renormalize))
