"""Root-mean-square norm behind the residual's addition: what stands in front of the attention and of the feed-forward
block of a decoder layer (RMSNorm, nsa/model/llama_dense.py:19-134).

    h = round(x + residual)        the stream, in the residual's dtype; h = x without a residual
    y = h / sqrt(mean(h^2) + eps) * weight

One kernel reads x and the residual once and writes h and y; fp32 inside, one rounding each.  `rms_norm_fp8` writes y as
fp8 with a scale per row, the operands of `linear_fp8`."""
from __future__ import annotations

import ctypes as C
from typing import Optional, Tuple, Union

import torch
from torch import Tensor

from . import _lib as L
from . import ops

_X = (torch.bfloat16, torch.float16, torch.float32)


def _check(x: Tensor, weight: Tensor, residual: Optional[Tensor], what: str) -> None:
    ops._need_cuda(x, weight, residual)
    ops._same_device(x, weight=weight, residual=residual)
    if x.dtype not in _X:
        raise TypeError(f"{what}: x must be bf16, fp16 or fp32, got {x.dtype}")
    if x.dim() < 1 or weight.shape != x.shape[-1:]:
        raise ValueError(f"{what}: weight shape {tuple(weight.shape)} does not match x {tuple(x.shape)}")
    if weight.dtype not in (x.dtype, torch.float32):
        raise TypeError(f"{what}: weight must have x's dtype or fp32, got {weight.dtype} beside {x.dtype}")
    if residual is not None:
        if residual.shape != x.shape:
            raise ValueError(f"{what}: residual shape {tuple(residual.shape)} does not match x {tuple(x.shape)}")
        if residual.dtype not in (x.dtype, torch.float32):
            raise TypeError(f"{what}: residual must have x's dtype or fp32, got {residual.dtype} beside {x.dtype}")


_plans = ops.Plans()


def _plan(x: Tensor, weight: Tensor, residual: Optional[Tensor], eps: float, y_dtype: Optional[torch.dtype], what: str) -> bytes:
    """nsa_norm_args without pointers, from checked operands; y_dtype None: x's."""
    key = (x.shape, x.dtype, x.device, weight.shape, weight.dtype, weight.device, eps, y_dtype,
           None if residual is None else (residual.shape, residual.dtype, residual.device))
    plan = _plans.get(key)
    if plan is None:
        _check(x, weight, residual, what)
        N, xc = x.shape[-1], L.dtype_code(x.dtype)
        a = L.NormArgs(rows=x.numel() // N if N else 0, hidden=N, x_dtype=xc, res_dtype=xc if residual is None else L.dtype_code(residual.dtype),
                       w_dtype=L.dtype_code(weight.dtype), y_dtype=xc if y_dtype is None else L.dtype_code(y_dtype), eps=eps)
        plan = _plans.keep(key, bytes(a))
    return plan


def _forward(plan: bytes, x: Tensor, weight: Tensor, residual: Optional[Tensor], y: Tensor, scale: Optional[Tensor], want_rstd: bool):
    """(h or None, rstd or None); dense operands."""
    a = L.NormArgs.from_buffer_copy(plan)
    a.x, a.weight, a.y = x.data_ptr(), weight.data_ptr(), y.data_ptr()
    h = rstd = None
    if residual is not None:
        h = torch.empty_like(residual)
        a.residual, a.h = residual.data_ptr(), h.data_ptr()
    if scale is not None:
        a.scale = scale.data_ptr()
    if want_rstd:
        rstd = x.new_empty(a.rows, dtype=torch.float32)
        a.rstd = rstd.data_ptr()
    L.call(L.load().nsa_rms_norm, a, x.get_device(), "nsa_rms_norm")
    return h, rstd


class _RmsNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, plan):
        y = torch.empty_like(x)
        h, rstd = _forward(plan, x, weight, residual, y, None, True)
        ctx.save_for_backward(x if h is None else h, weight, rstd)
        ctx.x_dtype, ctx.stream = x.dtype, residual is not None
        ctx.set_materialize_grads(False)
        return y if h is None else (y, h)

    @staticmethod
    @ops.first_order
    def backward(ctx, dy, dh=None):
        h, weight, rstd = ctx.saved_tensors
        dy = torch.zeros(h.shape, device=h.device, dtype=ctx.x_dtype) if dy is None else dy.contiguous()
        dh = None if dh is None else dh.contiguous()
        N = h.shape[-1]
        rows = h.numel() // N
        dx = torch.empty_like(dy)
        dres = torch.empty_like(h) if ctx.stream and h.dtype != ctx.x_dtype else None
        dw = torch.empty_like(weight) if ctx.needs_input_grad[2] else None
        lib = L.load()
        with L.on_device(h):
            need = lib.nsa_rms_norm_bwd_ws_bytes(rows, N)
        ws = h.new_empty(need, dtype=torch.uint8)
        a = L.NormBwdArgs(dy.data_ptr(), L.ptr(dh), h.data_ptr(), weight.data_ptr(), rstd.data_ptr(), dx.data_ptr(), L.ptr(dres), L.ptr(dw),
                          ws.data_ptr(), need, rows, N, L.dtype_code(ctx.x_dtype), L.dtype_code(h.dtype), L.dtype_code(weight.dtype))
        L.call(lib.nsa_rms_norm_bwd, a, h.get_device(), "nsa_rms_norm_bwd")
        # the same values reach x and the residual
        return dx, (dx if dres is None else dres) if ctx.stream else None, dw, None


def rms_norm(x: Tensor, weight: Tensor, *, residual: Optional[Tensor] = None, eps: float = 1e-6) -> Union[Tensor, Tuple[Tensor, Tensor]]:
    """x [..., N] bf16, fp16 or fp32, weight [N] (x's dtype or fp32), residual like x (x's dtype or fp32).
    Returns y in x's dtype; with a residual (y, h), h = x + residual being the new stream in the residual's dtype.
    Differentiable wrt x, residual and weight."""
    plan = _plan(x, weight, residual, float(eps), None, "rms_norm")
    x, weight = ops._dense(x, "x"), ops._dense(weight, "weight")
    if residual is not None:
        residual = ops._dense(residual, "residual")
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (residual is not None and residual.requires_grad)):
        return _RmsNormFn.apply(x, residual, weight, plan)
    y = torch.empty_like(x)
    h, _ = _forward(plan, x, weight, residual, y, None, False)
    return y if h is None else (y, h)


def rms_norm_fp8(x: Tensor, weight: Tensor, *, residual: Optional[Tensor] = None, eps: float = 1e-6,
                 fmt: torch.dtype = torch.float8_e4m3fn) -> Tuple[Tensor, ...]:
    """The same norm with an fp8 result: (q, scale) or, with a residual, (q, scale, h).  q [..., N] in `fmt`, scale [...] fp32
    per row: y ~= q * scale, scale = max(max|y|, 1e-12) / fmt_max.  Inference only."""
    if fmt not in ops._8:
        raise ValueError(f"unsupported fp8 format: {fmt}")
    plan = _plan(x, weight, residual, float(eps), fmt, "rms_norm_fp8")
    x, weight = ops._dense(x.detach(), "x"), ops._dense(weight.detach(), "weight")
    if residual is not None:
        residual = ops._dense(residual.detach(), "residual")
    q, scale = torch.empty_like(x, dtype=fmt), x.new_empty(x.shape[:-1], dtype=torch.float32)
    h, _ = _forward(plan, x, weight, residual, q, scale, False)
    return (q, scale) if h is None else (q, scale, h)


def quantize_rows_to_fp8(x: Tensor, *, fmt: torch.dtype = torch.float8_e4m3fn) -> Tuple[Tensor, Tensor]:
    """x [..., N] bf16, fp16 or fp32 -> (q in `fmt`, scale [...] fp32), a scale per row by the rule of `rms_norm_fp8`: the weights
    (and any activations) of `linear_fp8`."""
    if fmt not in ops._8:
        raise ValueError(f"unsupported fp8 format: {fmt}")
    ops._need_cuda(x)
    if x.dtype not in _X or x.dim() < 1:
        raise TypeError(f"quantize_rows_to_fp8: x must be a bf16, fp16 or fp32 tensor of rows, got {x.dtype}")
    x = ops._dense(x.detach(), "x")
    N = x.shape[-1]
    q = torch.empty(x.shape, device=x.device, dtype=fmt)
    scale = torch.empty(x.shape[:-1], device=x.device, dtype=torch.float32)
    with L.on_device(x):
        L.check(L.load().nsa_quantize_rows_fp8(x.data_ptr(), q.data_ptr(), scale.data_ptr(), scale.numel(), N, L.dtype_code(x.dtype),
                                               L.dtype_code(fmt), L.stream_ptr()), "nsa_quantize_rows_fp8")
    return q, scale


__all__ = ["rms_norm", "rms_norm_fp8", "quantize_rows_to_fp8"]
