"""Rotary embedding with several position axes (time, height and width of image and video tokens), from the projections'
token-major tensors to the attention's head-major ones: `rope_to_heads` of q, k and v in one launch, with the angles
formed from integer positions instead of read from tables, and with gradients.

Frequency j of D/2 turns by positions[axis(j), b, t] * inv_freq[j]; axis a owns sections[a] consecutive frequencies.
One axis is the ordinary rotary embedding (nsa/model/llama_dense.py:19-37) at arbitrary positions."""
from __future__ import annotations

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


def _heads(t: Tensor, name: str) -> Tensor:
    """`t` as the kernel reads it: heads and columns dense, the batch and token pitch anything (slices of a packed projection)."""
    if t.is_contiguous() or t.dim() != 4:
        return t
    _, _, head, col = t.stride()
    D = t.shape[3]
    return t if (col == 1 or D == 1) and (head == D or t.shape[2] == 1) else ops._dense(t, name)


def rope_axes_to_heads(q: Tensor, k: Tensor, v: Tensor, positions: Tensor, inv_freq: Tensor, sections: Sequence[int], *,
                       dtype: torch.dtype = torch.bfloat16) -> Tuple[Tensor, Tensor, Tensor]:
    """q [B,T,H,D], k and v [B,T,Hkv,D] as the projections leave them (one dtype: fp32, bf16 or fp16; slices of a packed
    projection are read where they lie), positions [axes,B,T] int32 or int64, inv_freq [D/2] (fp64; fp32 is converted),
    sections: frequencies of each axis, D/2 in all.  Returns q and k rotated, v as it is, [B,heads,T,D] in `dtype` (bf16 or
    fp16): fp32 inside, one rounding.  Differentiable wrt q, k and v."""
    if dtype not in ops._16:
        raise TypeError(f"rope_axes_to_heads: the result is bf16 or fp16, not {dtype}")
    if inv_freq.dtype == torch.float32:
        inv_freq = inv_freq.to(torch.float64)
    if not (q.is_contiguous() and k.is_contiguous() and v.is_contiguous() and positions.is_contiguous() and inv_freq.is_contiguous()):
        q, k, v = _heads(q, "q"), _heads(k, "k"), _heads(v, "v")
        positions, inv_freq = ops._dense(positions, "positions"), ops._dense(inv_freq, "inv_freq")
    return tuple(L.torch_ops().rope_axes(q, k, v, positions, inv_freq, sections, L.dtype_code(dtype)))


__all__ = ["rope_axes_to_heads", "rope_frequencies"]
