"""Rotary embedding with several position axes (time, height and width of image and video tokens), from the projections'
token-major tensors to the attention's head-major ones: `rope_to_heads` of q, k and v in one launch, with the angles
formed from integer positions instead of read from tables, and with gradients.

Frequency j of D/2 turns by positions[axis(j), b, t] * inv_freq[j]; axis a owns sections[a] consecutive frequencies.
One axis is the ordinary rotary embedding (nsa/model/llama_dense.py:19-37) at arbitrary positions."""
from __future__ import annotations

import ctypes as C
from typing import Sequence, Tuple

import torch
from torch import Tensor

from . import _lib as L
from . import ops


def rope_frequencies(head_dim: int, base: float = 10000.0, device="cuda") -> Tensor:
    """inv_freq [D/2] fp64: base ** (-2 j / D), the frequencies of `rope_cache`.  Scale or replace them freely."""
    if head_dim <= 0 or head_dim % 2:
        raise ValueError(f"rope_frequencies: head_dim {head_dim} must be even")
    return float(base) ** (-torch.arange(0, head_dim, 2, device=device, dtype=torch.float64) / head_dim)


def _pitched(t: Tensor) -> bool:
    """Heads and columns dense; the batch and token pitch may be anything (slices of a packed projection)."""
    D = t.shape[-1]
    _, _, head, col = t.stride()
    return (col == 1 or D == 1) and (head == D or t.shape[2] == 1)


def _check(q, k, v, positions, inv_freq, sections, dtype) -> Tuple[int, ...]:
    ops._need_cuda(q, k, v, positions, inv_freq)
    ops._same_device(q, k=k, v=v, positions=positions, inv_freq=inv_freq)
    if q.dim() != 4:
        raise ValueError(f"rope_axes_to_heads: q must be [B,T,H,D], got {tuple(q.shape)}")
    B, T, H, D = q.shape
    if k.dim() != 4 or k.shape[:2] != (B, T) or k.shape[3] != D or v.shape != k.shape:
        raise ValueError(f"rope_axes_to_heads: k/v shapes {tuple(k.shape)}/{tuple(v.shape)} do not match q {tuple(q.shape)}")
    if k.dtype != q.dtype or v.dtype != q.dtype or q.dtype not in (torch.float32, torch.bfloat16, torch.float16):
        raise TypeError("rope_axes_to_heads: q, k and v must share a dtype (fp32, bf16 or fp16)")
    if dtype not in ops._16:
        raise TypeError(f"rope_axes_to_heads: the result is bf16 or fp16, not {dtype}")
    sections = tuple(int(s) for s in sections)
    if D % 2 or not 1 <= len(sections) <= 8 or min(sections) < 0 or sum(sections) != D // 2:
        raise ValueError(f"rope_axes_to_heads: 1 to 8 sections that add up to D/2 = {D / 2:g} are needed, got {sections}")
    if positions.shape != (len(sections), B, T) or positions.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"rope_axes_to_heads: positions must be [{len(sections)},{B},{T}] int32 or int64, got {tuple(positions.shape)} {positions.dtype}")
    if inv_freq.shape != (D // 2,) or inv_freq.dtype not in (torch.float64, torch.float32):
        raise ValueError(f"rope_axes_to_heads: inv_freq must be [{D // 2}] fp64 or fp32, got {tuple(inv_freq.shape)} {inv_freq.dtype}")
    return sections


_plans = ops.Plans()


def _plan(q: Tensor, k: Tensor, v: Tensor, positions: Tensor, inv_freq: Tensor, sections: Sequence[int], dtype: torch.dtype) -> bytes:
    """nsa_rope_axes_args without pointers, from checked operands (the pitches of a packed projection included)."""
    sections = tuple(sections)
    key = (q.shape, k.shape, v.shape, q.dtype, k.dtype, v.dtype, q.device, k.device, v.device, q.stride(), k.stride(), v.stride(),
           positions.shape, positions.dtype, positions.device, inv_freq.shape, inv_freq.dtype, inv_freq.device, sections, dtype)
    plan = _plans.get(key)
    if plan is None:
        sections = _check(q, k, v, positions, inv_freq, sections, dtype)
        q, k, v = (t if _pitched(t) else torch.empty(t.shape, device="meta") for t in (q, k, v))     # what _dense makes of the others
        B, T, H, D = q.shape
        a = L.RopeAxesArgs(q_batch=q.stride(0), q_token=q.stride(1), k_batch=k.stride(0), k_token=k.stride(1), v_batch=v.stride(0), v_token=v.stride(1),
                           B=B, T=T, H=H, Hkv=k.shape[2], D=D, n_axes=len(sections), sections=(C.c_int32 * 8)(*sections),
                           pos64=int(positions.dtype == torch.int64), x_dtype=L.dtype_code(key[3]), y_dtype=L.dtype_code(dtype))
        plan = _plans.keep(key, bytes(a))
    return plan


def _launch(plan: bytes, src, dst, positions: Tensor, inv_freq: Tensor, backward: bool) -> None:
    a = L.RopeAxesArgs.from_buffer_copy(plan)
    a.q, a.k, a.v = src[0].data_ptr(), src[1].data_ptr(), src[2].data_ptr()
    a.q_out, a.k_out, a.v_out = dst[0].data_ptr(), dst[1].data_ptr(), dst[2].data_ptr()
    a.positions, a.inv_freq, a.backward = positions.data_ptr(), inv_freq.data_ptr(), backward
    L.call(L.load().nsa_rope_axes, a, positions.get_device(), "nsa_rope_axes")


def _forward(plan, q, k, v, positions, inv_freq, dtype):
    B, T, H, D = q.shape
    kv = (B, k.shape[2], T, D)
    out = q.new_empty((B, H, T, D), dtype=dtype), q.new_empty(kv, dtype=dtype), q.new_empty(kv, dtype=dtype)
    _launch(plan, (q, k, v), out, positions, inv_freq, False)
    return out


class _RopeAxesFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, positions, inv_freq, plan, dtype):
        ctx.save_for_backward(positions, inv_freq)
        ctx.plan, ctx.x_dtype = plan, q.dtype
        return _forward(plan, q, k, v, positions, inv_freq, dtype)

    @staticmethod
    @ops.first_order
    def backward(ctx, dq, dk, dv):
        B, H, T, D = dq.shape
        kv = (B, T, dk.shape[1], D)
        grads = dq.new_empty((B, T, H, D), dtype=ctx.x_dtype), dq.new_empty(kv, dtype=ctx.x_dtype), dq.new_empty(kv, dtype=ctx.x_dtype)
        _launch(ctx.plan, (dq.contiguous(), dk.contiguous(), dv.contiguous()), grads, *ctx.saved_tensors, True)
        return (*grads, None, None, None, None)


def rope_axes_to_heads(q: Tensor, k: Tensor, v: Tensor, positions: Tensor, inv_freq: Tensor, sections: Sequence[int], *,
                       dtype: torch.dtype = torch.bfloat16) -> Tuple[Tensor, Tensor, Tensor]:
    """q [B,T,H,D], k and v [B,T,Hkv,D] as the projections leave them (one dtype: fp32, bf16 or fp16; slices of a packed
    projection are read where they lie), positions [axes,B,T] int32 or int64, inv_freq [D/2] (fp64; fp32 is converted),
    sections: frequencies of each axis, D/2 in all.  Returns q and k rotated, v as it is, [B,heads,T,D] in `dtype` (bf16 or
    fp16): fp32 inside, one rounding.  Differentiable wrt q, k and v."""
    plan = _plan(q, k, v, positions, inv_freq, sections, dtype)
    q, k, v = (t if _pitched(t) else ops._dense(t, n) for t, n in ((q, "q"), (k, "k"), (v, "v")))
    positions = ops._dense(positions, "positions")
    if inv_freq.dtype != torch.float64 or not inv_freq.is_contiguous():
        inv_freq = inv_freq.to(torch.float64).contiguous()
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return _RopeAxesFn.apply(q, k, v, positions, inv_freq, plan, dtype)
    return _forward(plan, q, k, v, positions, inv_freq, dtype)


__all__ = ["rope_axes_to_heads", "rope_frequencies"]
