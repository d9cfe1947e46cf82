"""The caller of the NSA forward: the attention module between its projections.

Mirrors `NSAAttention.forward` of the reference (nsa/model/llama_nsa.py:67-96):

    q,k,v = proj(x).view(B,T,H,D).transpose(1,2); q,k = rope(q,k); gates = gate(x).view(B,T,H,3).permute(0,2,1,3)
    out = nsa_forward(q,k,v,cfg,gate_logits=gates); out = out.transpose(1,2).contiguous().view(B,T,H*D)

Between the projection GEMMs and `o_proj` the reference makes ten full-tensor passes (three transposes
to head-major, five element-wise kernels of the rotary embedding, the bf16 casts, the gate permute and
the transpose back).  Here each of q, k, v is read once and written once by `nsa_rope_to_heads`
(rotation in fp32, one rounding, head-major 16-bit result), the gate logits are read where they lie
([B,T,H,3]) and the kernel writes [B,T,H*D] directly.

`NSABlock` is the decoder layer around it (the reference's Llama block, nsa/model/llama_dense.py:19-134 with the attention of
nsa/model/llama_nsa.py:38-96), in 16 bits, for training, prefill and decoding: norm, projections, rotary embedding with any
number of position axes, attention, output projection with the residual in its epilogue, norm with the residual's
addition, gated feed-forward block with the residual in its epilogue.
"""
from __future__ import annotations

from typing import Dict, Optional, Sequence, Tuple

import torch
import torch.nn as nn
from torch import Tensor

from . import ops
from .decode import KVCache, nsa_decode
from .forward import _fused_forward, nsa_forward
from .norm import rms_norm
from .projections import gated_mlp, linear
from .rotary import rope_axes_to_heads, rope_frequencies


def rope_cache(seq_len: int, head_dim: int, base: float, device, dtype=torch.float32):
    """cos/sin tables [T, D] (`_build_rope_cache`, nsa/model/llama_dense.py:24-29)."""
    inv_freq = 1.0 / (base ** (torch.arange(0, head_dim, 2, device=device, dtype=torch.float32) / head_dim))
    t = torch.arange(seq_len, device=device, dtype=torch.float32)
    emb = torch.outer(t, inv_freq)
    emb = torch.cat((emb, emb), dim=-1)
    return emb.cos().to(dtype), emb.sin().to(dtype)


def nsa_attention_token_major(q: Tensor, k: Tensor, v: Tensor, cos: Optional[Tensor], sin: Optional[Tensor], cfg, *,
                              gate_logits: Optional[Tensor] = None, dtype: torch.dtype = torch.bfloat16,
                              pool_proj_k: Optional[Tensor] = None, pool_proj_v: Optional[Tensor] = None) -> Tensor:
    """q [B,T,H,D], k/v [B,T,Hkv,D] as the projections leave them (fp32, bf16 or fp16), cos/sin [T,D]
    (None: no rotary embedding), gate_logits [B,T,H,3] -> [B,T,H*D] in `dtype`.  Inference path (no autograd).
    pool_proj_k / pool_proj_v [block_size_c, D]: learned pooling (cfg.pool == "learned")."""
    B, T, H, D = q.shape
    qh = ops.rope_to_heads(q, cos, sin, dtype)
    kh = ops.rope_to_heads(k, cos, sin, dtype)
    vh = ops.rope_to_heads(v, None, None, dtype)
    scale = cfg.scale if cfg.scale is not None else 1.0 / (D ** 0.5)
    learned = getattr(cfg, "pool", "mean") == "learned"
    if learned and (pool_proj_k is None or pool_proj_v is None):
        raise ValueError("pool='learned' needs pool_proj_k and pool_proj_v")
    out = _fused_forward(qh, kh, vh, cfg, float(scale), getattr(cfg, "stride_c", None), gate_logits, None, 1.0, 1.0, 1.0,
                         token_major=True, pool_proj=(pool_proj_k, pool_proj_v) if learned else None)
    return out.view(B, T, H * D)


class NSAAttention(nn.Module):
    """Same parameters and forward signature as the reference's module (nsa/model/llama_nsa.py:38-96), so a
    state dict moves across unchanged; `n_kv_heads` < `n_heads` (grouped K/V) is an extension.
    Without autograd the token-major route above runs; with it, the reference's own sequence of
    steps around the differentiable `nsa_forward`."""

    def __init__(self, hidden_size: int, n_heads: int, head_dim: int, nsa_cfg, n_kv_heads: Optional[int] = None):
        super().__init__()
        self.n_heads, self.head_dim = n_heads, head_dim
        self.n_kv_heads = n_heads if n_kv_heads is None else n_kv_heads
        self.nsa_cfg = nsa_cfg
        # learned compressed-pool projections, as the reference module creates them (nsa/model/llama_nsa.py:59-65);
        # used by the inference route only -- training with pool="learned" is not provided
        if getattr(nsa_cfg, "pool", "mean") == "learned":
            self.pool_proj_k = nn.Parameter(torch.randn(int(nsa_cfg.block_size_c), head_dim) / head_dim ** 0.5)
            self.pool_proj_v = nn.Parameter(torch.randn(int(nsa_cfg.block_size_c), head_dim) / head_dim ** 0.5)
        else:
            self.pool_proj_k = self.pool_proj_v = None
        self.q_proj = nn.Linear(hidden_size, n_heads * head_dim, bias=False)
        self.k_proj = nn.Linear(hidden_size, self.n_kv_heads * head_dim, bias=False)
        self.v_proj = nn.Linear(hidden_size, self.n_kv_heads * head_dim, bias=False)
        self.o_proj = nn.Linear(n_heads * head_dim, hidden_size, bias=False)
        self.gate = nn.Linear(hidden_size, n_heads * 3, bias=False)

    def forward(self, x: Tensor, cos: Tensor, sin: Tensor) -> Tensor:
        B, T, _ = x.shape
        H, Hkv, D = self.n_heads, self.n_kv_heads, self.head_dim
        q = self.q_proj(x).view(B, T, H, D)
        k = self.k_proj(x).view(B, T, Hkv, D)
        v = self.v_proj(x).view(B, T, Hkv, D)
        gates = self.gate(x).view(B, T, H, 3)
        if not (torch.is_grad_enabled() and (x.requires_grad or any(p.requires_grad for p in self.parameters()))):
            out = nsa_attention_token_major(q, k, v, cos, sin, self.nsa_cfg, gate_logits=gates, pool_proj_k=self.pool_proj_k,
                                            pool_proj_v=self.pool_proj_v).to(x.dtype)
            return self.o_proj(out)
        q, k, v = (t.transpose(1, 2) for t in (q, k, v))
        c, s = cos[None, None], sin[None, None]
        rot = lambda t: torch.cat((-t[..., D // 2:], t[..., :D // 2]), dim=-1)
        q, k = q * c + rot(q) * s, k * c + rot(k) * s
        kd = torch.bfloat16
        out = nsa_forward(q.to(kd), k.to(kd), v.to(kd), self.nsa_cfg,
                          gate_logits=gates.permute(0, 2, 1, 3).contiguous().to(kd)).to(x.dtype)
        return self.o_proj(out.transpose(1, 2).contiguous().view(B, T, H * D))

    def attend(self, x: Tensor, positions: Tensor, inv_freq: Tensor, sections: Sequence[int], *, residual: Optional[Tensor] = None,
               cache: Optional[KVCache] = None) -> Tensor:
        """The module in bf16 or fp16 on the layer's own operators: x [B,T,hidden] -> [B,T,hidden] (+ residual, in the output
        projection's epilogue).  positions [axes,B,T], inv_freq and sections as for `rope_axes_to_heads`.  With `cache`
        (decoding, no gradients) the T positions are appended to it and attend everything it holds; else they attend each
        other.  Differentiable without a cache; pool="learned" takes the inference route without a cache only (a KVCache keeps
        window means)."""
        B, T, _ = x.shape
        H, Hkv, D = self.n_heads, self.n_kv_heads, self.head_dim
        cfg = self.nsa_cfg
        if cache is not None and getattr(cfg, "pool", "mean") == "learned":
            raise NotImplementedError("NSAAttention.attend: the cache keeps window means; pool='learned' has no decoding")
        q = linear(x, self.q_proj.weight).view(B, T, H, D)
        k = linear(x, self.k_proj.weight).view(B, T, Hkv, D)
        v = linear(x, self.v_proj.weight).view(B, T, Hkv, D)
        gates = linear(x, self.gate.weight).view(B, T, H, 3)
        q, k, v = rope_axes_to_heads(q, k, v, positions, inv_freq, sections, dtype=x.dtype)
        if cache is not None:
            if torch.is_grad_enabled() and any(t.requires_grad for t in (q, k, v, gates)):
                raise RuntimeError("NSAAttention.attend: a cached step has no gradients; call it under torch.no_grad()")
            cache.append(k, v)
            out = nsa_decode(q, cache, gate_logits=gates.permute(0, 2, 1, 3).contiguous()).transpose(1, 2).contiguous()
        elif torch.is_grad_enabled() and any(t.requires_grad for t in (q, k, v, gates)):
            out = nsa_forward(q, k, v, cfg, gate_logits=gates.permute(0, 2, 1, 3).contiguous()).transpose(1, 2).contiguous()
        else:
            learned = getattr(cfg, "pool", "mean") == "learned"
            scale = float(cfg.scale if cfg.scale is not None else D ** -0.5)
            out = _fused_forward(q, k, v, cfg, scale, getattr(cfg, "stride_c", None), gates, None, 1.0, 1.0, 1.0, token_major=True,
                                 pool_proj=(self.pool_proj_k, self.pool_proj_v) if learned else None)
        return linear(out.view(B, T, H * D), self.o_proj.weight, residual=residual)


class NSABlock(nn.Module):
    """A decoder layer in bf16 or fp16: x + attention(norm(x)), then + feed-forward(norm(.)).  `rope_sections`: frequencies of
    each position axis, head_dim / 2 in all (default: one axis)."""

    def __init__(self, hidden_size: int, n_heads: int, head_dim: int, nsa_cfg, intermediate_size: int, n_kv_heads: Optional[int] = None, *,
                 eps: float = 1e-6, activation: Optional[str] = "silu", rope_sections: Optional[Sequence[int]] = None, rope_base: float = 10000.0):
        super().__init__()
        self.attn = NSAAttention(hidden_size, n_heads, head_dim, nsa_cfg, n_kv_heads)
        self.attn_norm = nn.Parameter(torch.ones(hidden_size))
        self.mlp_norm = nn.Parameter(torch.ones(hidden_size))
        self.gate_proj = nn.Linear(hidden_size, intermediate_size, bias=False)
        self.up_proj = nn.Linear(hidden_size, intermediate_size, bias=False)
        self.down_proj = nn.Linear(intermediate_size, hidden_size, bias=False)
        self.eps, self.activation = eps, activation
        self.rope_sections = tuple(rope_sections) if rope_sections is not None else (head_dim // 2,)
        self.rope_base = rope_base
        # fp64, and stays that when the module is cast; by device and base, and kept while the module lives, since a captured
        # step or another stream's may still read an earlier one
        self._inv_freq: Dict[Tuple, Tensor] = {}

    def _frequencies(self, device: torch.device) -> Tensor:
        key = (device, float(self.rope_base), self.attn.head_dim)
        f = self._inv_freq.get(key)
        if f is not None:
            return f
        with torch.inference_mode(False):                    # a later training step saves it for its backward
            f = rope_frequencies(self.attn.head_dim, self.rope_base, device)
        if device.type == "cuda":
            with torch.cuda.device(device):
                if torch.cuda.is_current_stream_capturing():
                    return f                                 # holds nothing until the replay
                torch.cuda.current_stream().synchronize()    # whichever stream the next call is on finds it filled
            self._inv_freq[key] = f
        return f

    def new_cache(self, batch: int, max_len: int) -> KVCache:
        a = self.attn
        return KVCache(batch, a.n_kv_heads, a.head_dim, max_len, a.nsa_cfg, dtype=a.q_proj.weight.dtype, device=a.q_proj.weight.device)

    def forward(self, x: Tensor, positions: Optional[Tensor] = None, *, cache: Optional[KVCache] = None) -> Tensor:
        """x [B,T,hidden]; positions [axes,B,T] int32 or int64 (None, with one axis: 0..T-1, or the T positions behind what
        `cache` holds).  cache (decoding, under torch.no_grad()): the step's keys and values are appended to it."""
        B, T, _ = x.shape
        inv_freq = self._frequencies(x.device)
        if positions is None:
            if len(self.rope_sections) != 1:
                raise ValueError(f"NSABlock: {len(self.rope_sections)} position axes need positions")
            start = 0 if cache is None else cache.length
            positions = torch.arange(start, start + T, device=x.device).expand(1, B, T).contiguous()
        h = rms_norm(x, self.attn_norm, eps=self.eps)
        a = self.attn.attend(h, positions, inv_freq, self.rope_sections, cache=cache)
        h, x = rms_norm(a, self.mlp_norm, residual=x, eps=self.eps)
        return gated_mlp(h, self.gate_proj.weight, self.up_proj.weight, self.down_proj.weight, activation=self.activation, residual=x)


__all__ = ["NSAAttention", "NSABlock", "nsa_attention_token_major", "rope_cache"]
