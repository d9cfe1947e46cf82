"""Projections with their epilogue, and the gated feed-forward block of a decoder layer.

    linear      y = act(x w^T + bias) + residual            one matrix product, everything else in its epilogue
    gated_mlp   y = (act(x wg^T) * (x wu^T)) wd^T + residual    (SwiGLU, nsa/model/llama_dense.py:19-134)

`linear` is what `nn.Linear` (weight [out, in]) and the elementwise kernels behind it compute in several passes;
`gated_mlp` forms both inner products in one kernel that writes only the gated result.  Both have hand-written
backwards whose results repeat bit for bit."""
from __future__ import annotations

from typing import Optional

import torch
from torch import Tensor

from . import _lib as L
from . import ops


def linear(x: Tensor, weight: Tensor, bias: Optional[Tensor] = None, *, activation: Optional[str] = None,
           residual: Optional[Tensor] = None) -> Tensor:
    """act(x weight^T + bias) + residual.  x [..., K], weight [N, K], bias [N], residual [..., N], all bf16 or all fp16;
    activation None, "silu", "gelu_tanh" or "relu".  Returns [..., N] in x's dtype: fp32 sums and epilogue, one rounding.
    Differentiable wrt x, weight, bias and residual (act' is kept in 16 bits of its own for the backward, whose dy act' is
    rounded to x's dtype before the gradients' products)."""
    if not (x.is_contiguous() and weight.is_contiguous()):
        x, weight = ops._dense(x, "x"), ops._dense(weight, "weight")
    if bias is not None and not bias.is_contiguous():
        bias = ops._dense(bias, "bias")
    if residual is not None and not residual.is_contiguous():
        residual = ops._dense(residual, "residual")
    return L.torch_ops().linear(x, weight, bias, residual, ops.activation_code(activation))


def linear_fp8(x: Tensor, weight: Tensor, x_scale: Tensor, w_scale: Tensor, bias: Optional[Tensor] = None, *,
               activation: Optional[str] = None, residual: Optional[Tensor] = None, dtype: torch.dtype = torch.bfloat16) -> Tensor:
    """The same on fp8 operands: act((x weight^T) * x_scale * w_scale + bias) + residual.  x [..., K] and weight [N, K] both e4m3 or both
    e5m2, x_scale [...] and w_scale [N] fp32 (`rms_norm_fp8`, `quantize_rows_to_fp8`); bias, residual and the result in `dtype`
    (bf16 or fp16).  Inference only."""
    if dtype not in ops._16:
        raise TypeError(f"linear_fp8: the result is bf16 or fp16, not {dtype}")
    x, weight, x_scale, w_scale = ops._dense(x, "x"), ops._dense(weight, "weight"), ops._dense(x_scale, "x_scale"), ops._dense(w_scale, "w_scale")
    if bias is not None and not bias.is_contiguous():
        bias = ops._dense(bias, "bias")
    if residual is not None and not residual.is_contiguous():
        residual = ops._dense(residual, "residual")
    return L.torch_ops().linear_fp8(x, weight, x_scale, w_scale, bias, residual, ops.activation_code(activation), L.dtype_code(dtype))


def gated_mlp(x: Tensor, w_gate: Tensor, w_up: Tensor, w_down: Tensor, *, activation: Optional[str] = "silu",
              residual: Optional[Tensor] = None) -> Tensor:
    """(act(x w_gate^T) * (x w_up^T)) w_down^T + residual.  x and residual [..., N], w_gate and w_up [F, N], w_down [N, F], all bf16 or all
    fp16; activation as for `linear` (None: the plain product of the two).  fp32 sums; the gated product is rounded to x's
    dtype between the two matrix products, the result once.  Differentiable wrt every tensor (the gradients of the two inner
    products are rounded to x's dtype before the gradients' products, their factors kept in 24 bits)."""
    if not (x.is_contiguous() and w_gate.is_contiguous() and w_up.is_contiguous() and w_down.is_contiguous()):
        x, w_gate, w_up, w_down = ops._dense(x, "x"), ops._dense(w_gate, "w_gate"), ops._dense(w_up, "w_up"), ops._dense(w_down, "w_down")
    if residual is not None and not residual.is_contiguous():
        residual = ops._dense(residual, "residual")
    return L.torch_ops().gated_mlp(x, w_gate, w_up, w_down, residual, ops.activation_code(activation))


__all__ = ["linear", "linear_fp8", "gated_mlp"]
