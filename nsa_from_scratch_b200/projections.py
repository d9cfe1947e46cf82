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


def _run(a, ws_bytes, call, what: str, like: Tensor) -> None:
    """One library call with the workspace that it asks for; every pointer of `a` is set."""
    index = like.get_device()
    if index != torch._C._cuda_getDevice():
        with torch.cuda.device(index):
            return _run(a, ws_bytes, call, what, like)
    need = ws_bytes(C.byref(a))
    if need:
        if need < 0:
            L.check(int(need), what)
        ws = like.new_empty(need, dtype=torch.uint8)
        a.ws, a.ws_bytes = ws.data_ptr(), need
    L.call(call, a, index, what)


def _check_rows(t: Optional[Tensor], name: str, shape, dtype, what: str) -> None:
    if t is not None and (t.shape != shape or t.dtype != dtype):
        raise ValueError(f"{what}: {name} must be {list(shape)} {dtype}, got {tuple(t.shape)} {t.dtype}")


def _meta(*ts: Optional[Tensor]):
    return tuple(None if t is None else (t.shape, t.dtype, t.device) for t in ts)


_plans = ops.Plans()


def _linear(plan: bytes, x: Tensor, w: Tensor, bias, residual, xs, ws, dtype: torch.dtype, want_slope: bool):
    """(y, slope or None); dense operands."""
    a = L.LinearArgs.from_buffer_copy(plan)
    y = x.new_empty((*x.shape[:-1], a.N), dtype=dtype)
    a.x, a.w, a.y = x.data_ptr(), w.data_ptr(), y.data_ptr()
    if bias is not None:
        a.bias = bias.data_ptr()
    if residual is not None:
        a.residual = residual.data_ptr()
    if xs is not None:
        a.x_scale, a.w_scale = xs.data_ptr(), ws.data_ptr()
    slope = None
    if want_slope:
        slope = torch.empty_like(y, dtype=torch.int16)
        a.slope = slope.data_ptr()
    lib = L.load()
    _run(a, lib.nsa_linear_ws_bytes, lib.nsa_linear, "nsa_linear", x)
    return y, slope


class _LinearFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, bias, residual, act, plan):
        y, slope = _linear(plan, x, w, bias, residual, None, None, x.dtype, act != 0 and any(ctx.needs_input_grad[:3]))
        ctx.save_for_backward(x, w, slope)
        return y

    @staticmethod
    @ops.first_order
    def backward(ctx, dy):
        x, w, slope = ctx.saved_tensors
        dy = dy.contiguous()
        N, K = w.shape
        want_x, want_w, want_b, want_r = ctx.needs_input_grad[:4]
        dx = torch.empty_like(x) if want_x else None
        dw = torch.empty_like(w) if want_w else None
        db = x.new_empty(N) if want_b else None
        if want_x or want_w or want_b:
            a = L.LinearBwdArgs(dy.data_ptr(), x.data_ptr(), w.data_ptr(), L.ptr(slope), L.ptr(dx), L.ptr(dw), L.ptr(db), None, 0, x.numel() // K, N, K,
                                L.dtype_code(x.dtype), slope is not None)
            lib = L.load()
            _run(a, lib.nsa_linear_bwd_ws_bytes, lib.nsa_linear_bwd, "nsa_linear_bwd", x)
        return dx, dw, db, dy if want_r else None, None, None


def linear(x: Tensor, weight: Tensor, bias: Optional[Tensor] = None, *, activation: Optional[str] = None,
           residual: Optional[Tensor] = None) -> Tensor:
    """act(x weight^T + bias) + residual.  x [..., K], weight [N, K], bias [N], residual [..., N], all bf16 or all fp16;
    activation None, "silu", "gelu_tanh" or "relu".  Returns [..., N] in x's dtype: fp32 sums and epilogue, one rounding.
    Differentiable wrt x, weight, bias and residual (act' is kept in 16 bits of its own for the backward)."""
    key = ("linear", activation, *_meta(x, weight, bias, residual))
    plan = _plans.get(key)
    if plan is None:
        ops._need_cuda(x, weight, bias, residual)
        ops._same_device(x, weight=weight, bias=bias, residual=residual)
        act = ops.activation_code(activation)
        if x.dtype not in ops._16 or weight.dtype != x.dtype:
            raise TypeError(f"linear: x and weight must both be bf16 or both fp16, got {x.dtype} and {weight.dtype}")
        if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1] or 0 in weight.shape:
            raise ValueError(f"linear: x {tuple(x.shape)} does not match weight {tuple(weight.shape)}")
        _check_rows(bias, "bias", weight.shape[:1], x.dtype, "linear")
        _check_rows(residual, "residual", (*x.shape[:-1], weight.shape[0]), x.dtype, "linear")
        code = L.dtype_code(x.dtype)
        N, K = weight.shape
        plan = _plans.keep(key, (bytes(L.LinearArgs(M=x.numel() // K, N=N, K=K, dtype=code, y_dtype=code, act=act)), act))
    x, weight = ops._dense(x, "x"), ops._dense(weight, "weight")
    if bias is not None:
        bias = ops._dense(bias, "bias")
    if residual is not None:
        residual = ops._dense(residual, "residual")
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad)
                                    or (residual is not None and residual.requires_grad)):
        return _LinearFn.apply(x, weight, bias, residual, plan[1], plan[0])
    return _linear(plan[0], x, weight, bias, residual, None, None, x.dtype, False)[0]


def linear_fp8(x: Tensor, weight: Tensor, x_scale: Tensor, w_scale: Tensor, bias: Optional[Tensor] = None, *,
               activation: Optional[str] = None, residual: Optional[Tensor] = None, dtype: torch.dtype = torch.bfloat16) -> Tensor:
    """The same on fp8 operands: act((x weight^T) * x_scale * w_scale + bias) + residual.  x [..., K] and weight [N, K] both e4m3 or both
    e5m2, x_scale [...] and w_scale [N] fp32 (`rms_norm_fp8`, `quantize_rows_to_fp8`); bias, residual and the result in `dtype`
    (bf16 or fp16).  Inference only."""
    key = ("linear_fp8", activation, dtype, *_meta(x, weight, x_scale, w_scale, bias, residual))
    plan = _plans.get(key)
    if plan is None:
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
        N, K = weight.shape
        plan = _plans.keep(key, bytes(L.LinearArgs(M=x.numel() // K, N=N, K=K, dtype=L.dtype_code(x.dtype), y_dtype=L.dtype_code(dtype), act=act)))
    x, weight, x_scale, w_scale = ops._dense(x, "x"), ops._dense(weight, "weight"), ops._dense(x_scale, "x_scale"), ops._dense(w_scale, "w_scale")
    if bias is not None:
        bias = ops._dense(bias, "bias")
    if residual is not None:
        residual = ops._dense(residual, "residual")
    return _linear(plan, x, weight, bias, residual, x_scale, w_scale, dtype, False)[0]


def _mlp(plan: bytes, x, wg, wu, wd, residual, keep):
    """(y, kept): dense operands; kept is () or, for the backward, act(g) and act'(g) * u in 24 bits (three tensors)
    and act(g) * u, rows padded to a multiple of 8."""
    a = L.GatedMlpArgs.from_buffer_copy(plan)
    y = torch.empty_like(x)
    a.x, a.wg, a.wu, a.wd, a.y = x.data_ptr(), wg.data_ptr(), wu.data_ptr(), wd.data_ptr(), y.data_ptr()
    if residual is not None:
        a.residual = residual.data_ptr()
    kept = ()
    if keep:
        shape = (a.M, (a.F + 7) // 8 * 8)
        kept = p, s, low, h = *(x.new_empty(shape, dtype=torch.int16) for _ in range(3)), x.new_empty(shape)
        a.p, a.s, a.low, a.h = p.data_ptr(), s.data_ptr(), low.data_ptr(), h.data_ptr()
    lib = L.load()
    _run(a, lib.nsa_gated_mlp_ws_bytes, lib.nsa_gated_mlp, "nsa_gated_mlp", x)
    return y, kept


class _GatedMlpFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, wg, wu, wd, residual, plan):
        y, kept = _mlp(plan, x, wg, wu, wd, residual, any(ctx.needs_input_grad[:4]))
        ctx.save_for_backward(x, wg, wu, wd, *kept)
        return y

    @staticmethod
    @ops.first_order
    def backward(ctx, dy):
        x, wg, wu, wd, *kept = ctx.saved_tensors
        dy = dy.contiguous()
        F, N = wg.shape
        M = x.numel() // N
        grads = [torch.empty_like(t) if want else None for t, want in zip((x, wg, wu, wd), ctx.needs_input_grad)]
        if any(ctx.needs_input_grad[:4]):
            a = L.GatedMlpBwdArgs(dy.data_ptr(), x.data_ptr(), wg.data_ptr(), wu.data_ptr(), wd.data_ptr(), *(t.data_ptr() for t in kept),
                                  *(L.ptr(t) for t in grads), None, 0, M, N, F, L.dtype_code(x.dtype))
            lib = L.load()
            _run(a, lib.nsa_gated_mlp_bwd_ws_bytes, lib.nsa_gated_mlp_bwd, "nsa_gated_mlp_bwd", x)
        return (*grads, dy if ctx.needs_input_grad[4] else None, None)


def gated_mlp(x: Tensor, w_gate: Tensor, w_up: Tensor, w_down: Tensor, *, activation: Optional[str] = "silu",
              residual: Optional[Tensor] = None) -> Tensor:
    """(act(x w_gate^T) * (x w_up^T)) w_down^T + residual.  x and residual [..., N], w_gate and w_up [F, N], w_down [N, F], all bf16 or all
    fp16; activation as for `linear` (None: the plain product of the two).  fp32 sums; the gated product is rounded to x's
    dtype between the two matrix products, the result once.  Differentiable wrt every tensor."""
    key = ("gated_mlp", activation, *_meta(x, w_gate, w_up, w_down, residual))
    plan = _plans.get(key)
    if plan is None:
        ops._need_cuda(x, w_gate, w_up, w_down, residual)
        ops._same_device(x, w_gate=w_gate, w_up=w_up, w_down=w_down, residual=residual)
        act = ops.activation_code(activation)
        if x.dtype not in ops._16 or any(w.dtype != x.dtype for w in (w_gate, w_up, w_down)):
            raise TypeError(f"gated_mlp: x and the weights must all be bf16 or all fp16, got {x.dtype}, {w_gate.dtype}, {w_up.dtype}, {w_down.dtype}")
        if (w_gate.dim() != 2 or x.dim() < 1 or x.shape[-1] != w_gate.shape[1] or w_up.shape != w_gate.shape or w_down.shape != w_gate.shape[::-1]
                or 0 in w_gate.shape):
            raise ValueError(f"gated_mlp: x {tuple(x.shape)} and weights {tuple(w_gate.shape)}, {tuple(w_up.shape)}, {tuple(w_down.shape)} do not match")
        _check_rows(residual, "residual", x.shape, x.dtype, "gated_mlp")
        F, N = w_gate.shape
        plan = _plans.keep(key, bytes(L.GatedMlpArgs(M=x.numel() // N, N=N, F=F, dtype=L.dtype_code(x.dtype), act=act)))
    x, w_gate, w_up, w_down = ops._dense(x, "x"), ops._dense(w_gate, "w_gate"), ops._dense(w_up, "w_up"), ops._dense(w_down, "w_down")
    if residual is not None:
        residual = ops._dense(residual, "residual")
    if torch.is_grad_enabled() and (x.requires_grad or w_gate.requires_grad or w_up.requires_grad or w_down.requires_grad
                                    or (residual is not None and residual.requires_grad)):
        return _GatedMlpFn.apply(x, w_gate, w_up, w_down, residual, plan)
    return _mlp(plan, x, w_gate, w_up, w_down, residual, False)[0]


__all__ = ["linear", "linear_fp8", "gated_mlp"]
