"""Projections with their epilogue, and the gated feed-forward block of a decoder layer.

    linear      y = act(x w^T + bias) + residual            one matrix product, everything else in its epilogue
    gated_mlp   y = (act(x wg^T) * (x wu^T)) wd^T + residual    (SwiGLU, nsa/model/llama_dense.py:19-134)

`linear` is what `nn.Linear` (weight [out, in]) and the elementwise kernels behind it compute in several passes;
`gated_mlp` forms both inner products in one kernel that writes only the gated result.  Both have hand-written
backwards whose results repeat bit for bit."""
from __future__ import annotations

import ctypes as C
from typing import Optional

import torch
from torch import Tensor

from . import _lib as L
from . import ops


def _ws(need: int, what: str, device) -> Optional[Tensor]:
    if need < 0:
        L.check(int(need), what)
    return torch.empty(need, device=device, dtype=torch.uint8) if need else None


def _check_rows(t: Optional[Tensor], name: str, shape, dtype, what: str) -> None:
    if t is not None and (t.shape != shape or t.dtype != dtype):
        raise ValueError(f"{what}: {name} must be {list(shape)} {dtype}, got {tuple(t.shape)} {t.dtype}")


def _linear(x: Tensor, w: Tensor, bias, residual, xs, ws_, act: int, dtype: torch.dtype, want_z: bool):
    """(y, z or None); dense operands."""
    N, K = w.shape
    lead = x.shape[:-1]
    M = x.numel() // K
    y = torch.empty((*lead, N), device=x.device, dtype=dtype)
    z = torch.empty((M, N), device=x.device, dtype=dtype) if want_z else None
    a = L.LinearArgs(x.data_ptr(), w.data_ptr(), L.ptr(bias), L.ptr(residual), L.ptr(xs), L.ptr(ws_), y.data_ptr(), L.ptr(z), None, 0,
                     M, N, K, L.dtype_code(x.dtype), L.dtype_code(dtype), act)
    lib = L.load()
    with L.on_device(x):
        need = lib.nsa_linear_ws_bytes(C.byref(a))
        ws = _ws(need, "nsa_linear", x.device)
        if ws is not None:
            a.ws, a.ws_bytes = ws.data_ptr(), need
        L.check(lib.nsa_linear(C.byref(a), L.stream_ptr()), "nsa_linear")
    return y, z


class _LinearFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, bias, residual, act):
        y, z = _linear(x, w, bias, residual, None, None, act, x.dtype, act != 0 and any(ctx.needs_input_grad[:3]))
        ctx.save_for_backward(x, w, z)
        ctx.act = act
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, w, z = ctx.saved_tensors
        dy = dy.contiguous()
        N, K = w.shape
        M = x.numel() // K
        want_x, want_w, want_b, want_r = ctx.needs_input_grad[:4]
        dx = torch.empty_like(x) if want_x else None
        dw = torch.empty_like(w) if want_w else None
        db = torch.empty(N, device=x.device, dtype=x.dtype) if want_b else None
        if want_x or want_w or want_b:
            a = L.LinearBwdArgs(dy.data_ptr(), x.data_ptr(), w.data_ptr(), L.ptr(z), L.ptr(dx), L.ptr(dw), L.ptr(db), None, 0, M, N, K,
                                L.dtype_code(x.dtype), ctx.act)
            lib = L.load()
            with L.on_device(x):
                need = lib.nsa_linear_bwd_ws_bytes(C.byref(a))
                ws = _ws(need, "nsa_linear_bwd", x.device)
                if ws is not None:
                    a.ws, a.ws_bytes = ws.data_ptr(), need
                L.check(lib.nsa_linear_bwd(C.byref(a), L.stream_ptr()), "nsa_linear_bwd")
        return dx, dw, db, dy if want_r else None, None


def linear(x: Tensor, weight: Tensor, bias: Optional[Tensor] = None, *, activation: Optional[str] = None,
           residual: Optional[Tensor] = None) -> Tensor:
    """act(x weight^T + bias) + residual.  x [..., K], weight [N, K], bias [N], residual [..., N], all bf16 or all fp16;
    activation None, "silu", "gelu_tanh" or "relu".  Returns [..., N] in x's dtype: fp32 sums and epilogue, one rounding.
    Differentiable wrt x, weight, bias and residual (act's argument is kept in x's dtype for the backward)."""
    ops._need_cuda(x, weight, bias, residual)
    ops._same_device(x, weight=weight, bias=bias, residual=residual)
    act = ops.activation_code(activation)
    if x.dtype not in ops._16 or weight.dtype != x.dtype:
        raise TypeError(f"linear: x and weight must both be bf16 or both fp16, got {x.dtype} and {weight.dtype}")
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1] or 0 in weight.shape:
        raise ValueError(f"linear: x {tuple(x.shape)} does not match weight {tuple(weight.shape)}")
    _check_rows(bias, "bias", weight.shape[:1], x.dtype, "linear")
    _check_rows(residual, "residual", (*x.shape[:-1], weight.shape[0]), x.dtype, "linear")
    x, weight = ops._dense(x, "x"), ops._dense(weight, "weight")
    bias = None if bias is None else ops._dense(bias, "bias")
    residual = None if residual is None else ops._dense(residual, "residual")
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias, residual)):
        return _LinearFn.apply(x, weight, bias, residual, act)
    return _linear(x, weight, bias, residual, None, None, act, x.dtype, False)[0]


def linear_fp8(x: Tensor, weight: Tensor, x_scale: Tensor, w_scale: Tensor, bias: Optional[Tensor] = None, *,
               activation: Optional[str] = None, residual: Optional[Tensor] = None, dtype: torch.dtype = torch.bfloat16) -> Tensor:
    """The same on fp8 operands: act((x weight^T) * x_scale * w_scale + bias) + residual.  x [..., K] and weight [N, K] both e4m3 or both
    e5m2, x_scale [...] and w_scale [N] fp32 (`rms_norm_fp8`, `quantize_rows_to_fp8`); bias, residual and the result in `dtype`
    (bf16 or fp16).  Inference only."""
    ops._need_cuda(x, weight, x_scale, w_scale, bias, residual)
    ops._same_device(x, weight=weight, x_scale=x_scale, w_scale=w_scale, bias=bias, residual=residual)
    act = ops.activation_code(activation)
    if x.dtype not in ops._8 or weight.dtype != x.dtype:
        raise TypeError(f"linear_fp8: x and weight must share an fp8 dtype, got {x.dtype} and {weight.dtype}")
    if dtype not in ops._16:
        raise TypeError(f"linear_fp8: the result is bf16 or fp16, not {dtype}")
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1] or 0 in weight.shape:
        raise ValueError(f"linear_fp8: x {tuple(x.shape)} does not match weight {tuple(weight.shape)}")
    _check_rows(x_scale, "x_scale", x.shape[:-1], torch.float32, "linear_fp8")
    _check_rows(w_scale, "w_scale", weight.shape[:1], torch.float32, "linear_fp8")
    _check_rows(bias, "bias", weight.shape[:1], dtype, "linear_fp8")
    _check_rows(residual, "residual", (*x.shape[:-1], weight.shape[0]), dtype, "linear_fp8")
    x, weight, x_scale, w_scale = (ops._dense(t.detach(), n) for t, n in ((x, "x"), (weight, "weight"), (x_scale, "x_scale"), (w_scale, "w_scale")))
    bias = None if bias is None else ops._dense(bias.detach(), "bias")
    residual = None if residual is None else ops._dense(residual.detach(), "residual")
    return _linear(x, weight, bias, residual, x_scale, w_scale, act, dtype, False)[0]


def _mlp(x, wg, wu, wd, residual, act, keep):
    """(y, g or None, u or None); dense operands."""
    F, N = wg.shape
    M = x.numel() // N
    y = torch.empty_like(x)
    g, u = (torch.empty((M, F), device=x.device, dtype=x.dtype) for _ in range(2)) if keep else (None, None)
    a = L.GatedMlpArgs(x.data_ptr(), wg.data_ptr(), wu.data_ptr(), wd.data_ptr(), L.ptr(residual), y.data_ptr(), L.ptr(g), L.ptr(u), None, 0,
                       M, N, F, L.dtype_code(x.dtype), act)
    lib = L.load()
    with L.on_device(x):
        need = lib.nsa_gated_mlp_ws_bytes(C.byref(a))
        ws = _ws(need, "nsa_gated_mlp", x.device)
        if ws is not None:
            a.ws, a.ws_bytes = ws.data_ptr(), need
        L.check(lib.nsa_gated_mlp(C.byref(a), L.stream_ptr()), "nsa_gated_mlp")
    return y, g, u


class _GatedMlpFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, wg, wu, wd, residual, act):
        y, g, u = _mlp(x, wg, wu, wd, residual, act, any(ctx.needs_input_grad[:4]))
        ctx.save_for_backward(x, wg, wu, wd, g, u)
        ctx.act = act
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, wg, wu, wd, g, u = ctx.saved_tensors
        dy = dy.contiguous()
        F, N = wg.shape
        M = x.numel() // N
        grads = [torch.empty_like(t) if want else None for t, want in zip((x, wg, wu, wd), ctx.needs_input_grad)]
        if any(ctx.needs_input_grad[:4]):
            a = L.GatedMlpBwdArgs(dy.data_ptr(), x.data_ptr(), wg.data_ptr(), wu.data_ptr(), wd.data_ptr(), g.data_ptr(), u.data_ptr(),
                                  *(L.ptr(t) for t in grads), None, 0, M, N, F, L.dtype_code(x.dtype), ctx.act)
            lib = L.load()
            with L.on_device(x):
                need = lib.nsa_gated_mlp_bwd_ws_bytes(C.byref(a))
                ws = _ws(need, "nsa_gated_mlp_bwd", x.device)
                if ws is not None:
                    a.ws, a.ws_bytes = ws.data_ptr(), need
                L.check(lib.nsa_gated_mlp_bwd(C.byref(a), L.stream_ptr()), "nsa_gated_mlp_bwd")
        return (*grads, dy if ctx.needs_input_grad[4] else None, None)


def gated_mlp(x: Tensor, w_gate: Tensor, w_up: Tensor, w_down: Tensor, *, activation: Optional[str] = "silu",
              residual: Optional[Tensor] = None) -> Tensor:
    """(act(x w_gate^T) * (x w_up^T)) w_down^T + residual.  x and residual [..., N], w_gate and w_up [F, N], w_down [N, F], all bf16 or all
    fp16; activation as for `linear` (None: the plain product of the two).  fp32 sums; the gated product is rounded to x's
    dtype between the two matrix products, the result once.  Differentiable wrt every tensor."""
    ops._need_cuda(x, w_gate, w_up, w_down, residual)
    ops._same_device(x, w_gate=w_gate, w_up=w_up, w_down=w_down, residual=residual)
    act = ops.activation_code(activation)
    if x.dtype not in ops._16 or any(w.dtype != x.dtype for w in (w_gate, w_up, w_down)):
        raise TypeError(f"gated_mlp: x and the weights must all be bf16 or all fp16, got {x.dtype}, {w_gate.dtype}, {w_up.dtype}, {w_down.dtype}")
    if w_gate.dim() != 2 or x.dim() < 1 or x.shape[-1] != w_gate.shape[1] or w_up.shape != w_gate.shape or w_down.shape != w_gate.shape[::-1] or 0 in w_gate.shape:
        raise ValueError(f"gated_mlp: x {tuple(x.shape)} and weights {tuple(w_gate.shape)}, {tuple(w_up.shape)}, {tuple(w_down.shape)} do not match")
    _check_rows(residual, "residual", x.shape, x.dtype, "gated_mlp")
    x, w_gate, w_up, w_down = (ops._dense(t, n) for t, n in ((x, "x"), (w_gate, "w_gate"), (w_up, "w_up"), (w_down, "w_down")))
    residual = None if residual is None else ops._dense(residual, "residual")
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, w_gate, w_up, w_down, residual)):
        return _GatedMlpFn.apply(x, w_gate, w_up, w_down, residual, act)
    return _mlp(x, w_gate, w_up, w_down, residual, act, False)[0]


__all__ = ["linear", "linear_fp8", "gated_mlp"]
