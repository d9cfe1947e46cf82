"""Root-mean-square norm behind the residual's addition: what stands in front of the attention and of the feed-forward
block of a decoder layer (RMSNorm, nsa/model/llama_dense.py:19-134).

    h = round(x + residual)        the stream, in the residual's dtype; h = x without a residual
    y = h / sqrt(mean(h^2) + eps) * weight

One kernel reads x and the residual once and writes h and y; fp32 inside, one rounding each.  `rms_norm_fp8` writes y as
fp8 with a scale per row, the operands of `linear_fp8`."""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch
from torch import Tensor

from . import _lib as L
from . import ops


def rms_norm(x: Tensor, weight: Tensor, *, residual: Optional[Tensor] = None, eps: float = 1e-6) -> Union[Tensor, Tuple[Tensor, Tensor]]:
    """x [..., N] bf16, fp16 or fp32, weight [N] (x's dtype or fp32), residual like x (x's dtype or fp32).
    Returns y in x's dtype; with a residual (y, h), h = x + residual being the new stream in the residual's dtype.
    Differentiable wrt x, residual and weight."""
    if not (x.is_contiguous() and weight.is_contiguous()):
        x, weight = ops._dense(x, "x"), ops._dense(weight, "weight")
    if residual is not None and not residual.is_contiguous():
        residual = ops._dense(residual, "residual")
    out = L.torch_ops().rms_norm(x, weight, residual, eps)
    return out[0] if residual is None else (out[0], out[1])


def rms_norm_fp8(x: Tensor, weight: Tensor, *, residual: Optional[Tensor] = None, eps: float = 1e-6,
                 fmt: torch.dtype = torch.float8_e4m3fn) -> Tuple[Tensor, ...]:
    """The same norm with an fp8 result: (q, scale) or, with a residual, (q, scale, h).  q [..., N] in `fmt`, scale [...] fp32
    per row: y ~= q * scale, scale = max(max|y|, 1e-12) / fmt_max.  Inference only."""
    if fmt not in ops._8:
        raise ValueError(f"unsupported fp8 format: {fmt}")
    if not (x.is_contiguous() and weight.is_contiguous()):
        x, weight = ops._dense(x, "x"), ops._dense(weight, "weight")
    if residual is not None and not residual.is_contiguous():
        residual = ops._dense(residual, "residual")
    return tuple(L.torch_ops().rms_norm_fp8(x, weight, residual, eps, L.dtype_code(fmt)))


def quantize_rows_to_fp8(x: Tensor, *, fmt: torch.dtype = torch.float8_e4m3fn) -> Tuple[Tensor, Tensor]:
    """x [..., N] bf16, fp16 or fp32 -> (q in `fmt`, scale [...] fp32), a scale per row by the rule of `rms_norm_fp8`: the weights
    (and any activations) of `linear_fp8`."""
    if fmt not in ops._8:
        raise ValueError(f"unsupported fp8 format: {fmt}")
    return tuple(L.torch_ops().quantize_rows(ops._dense(x, "x"), L.dtype_code(fmt)))


__all__ = ["rms_norm", "rms_norm_fp8", "quantize_rows_to_fp8"]
