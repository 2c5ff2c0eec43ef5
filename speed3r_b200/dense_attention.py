"""Dense attention inside each view, drop-in for the reference's ``FlashAttentionRope`` (the frame blocks of its decoder).

``FlashAttentionRope`` keeps the constructor signature, sub-module names (``qkv``, ``proj``, ``q_norm``, ``k_norm``) and ``forward(x, attn_bias=None,
xpos=None)`` of pi3/models/layers/attention.py:324-348, so that ``BlockRope(attn_class=FlashAttentionRope)`` loads a checkpoint unchanged.  Its
projections are ``ops.linear``; the split of the packed projection, the norms of every head of q and k and the rotary embedding are
``ops.qkv_norm_rope``, one pass with gradients; the attention itself stays PyTorch's ``scaled_dot_product_attention``, as in the reference.
"""
from __future__ import annotations

from typing import Optional

import torch
from torch import Tensor, nn

from . import ops
from .block import product_type
from .sparse_attention import RoPE2D, _global_hooks, _is_rope2d, _plain_rope, _TableRows, _watched, rope_tables


class FlashAttentionRope(nn.Module):
    def __init__(
        self,
        dim: int,
        num_heads: int = 8,
        qkv_bias: bool = False,
        proj_bias: bool = True,
        attn_drop: float = 0.0,
        proj_drop: float = 0.0,
        qk_norm: bool = False,
        norm_layer: nn.Module = nn.LayerNorm,
        rope=None,
    ) -> None:
        super().__init__()
        self.num_heads = num_heads
        head_dim = dim // num_heads
        self.scale = head_dim ** -0.5
        self.qkv = nn.Linear(dim, dim * 3, bias=qkv_bias)
        self.attn_drop = nn.Dropout(attn_drop)
        self.proj = nn.Linear(dim, dim, bias=proj_bias)
        self.proj_drop = nn.Dropout(proj_drop)
        self.q_norm = norm_layer(head_dim) if qk_norm else nn.Identity()
        self.k_norm = norm_layer(head_dim) if qk_norm else nn.Identity()
        self.rope = rope
        self._rows = _TableRows()    # table length when the rotary module is the reference's own

    @staticmethod
    def _linear(m: nn.Module, x: Tensor) -> Tensor:
        t = product_type(x, m)
        return m(x) if t is None else ops.linear(x.to(t), m.weight.to(t), m.bias)

    def _norms(self, d: int):
        """(kind, q_norm, k_norm) as ``ops.qkv_norm_rope`` takes them, None for other norms."""
        q, k = self.q_norm, self.k_norm
        if _watched(q) or _watched(k) or type(q) is not type(k):
            return None
        if type(q) is nn.Identity:
            return "layer", None, None
        if type(q) is nn.LayerNorm and tuple(q.normalized_shape) == tuple(k.normalized_shape) == (d,):
            return "layer", (q.weight, q.bias, q.eps), (k.weight, k.bias, k.eps)
        if type(q) is nn.RMSNorm and tuple(q.normalized_shape) == tuple(k.normalized_shape) == (d,) and q.eps is not None and k.eps is not None:
            return "rms", (q.weight, None, q.eps), (k.weight, None, k.eps)
        return None

    def _heads(self, qkv: Tensor, xpos: Optional[Tensor], B: int, N: int, d: int):
        """q, k and v [B, H, N, d]"""
        H, norms = self.num_heads, self._norms(d)
        turned = xpos is not None and self.rope is not None
        if (qkv.is_cuda and qkv.dtype in ops.NORM_TYPES and norms is not None and not _global_hooks() and d % 2 == 0 and d <= 256 and
                (not turned or (d % 4 == 0 and _is_rope2d(self.rope) and _plain_rope(self.rope)))):
            pos = cos = sin = None
            if turned:
                rows = self.rope._seq_len(xpos) if isinstance(self.rope, RoPE2D) else self._rows(xpos)
                cos, sin = rope_tables(self.rope, d // 2, rows, qkv.device, qkv.dtype)
                pos, cos, sin = xpos, cos[:, :d // 4], sin[:, :d // 4]                 # both halves of a row are alike
            return ops.qkv_norm_rope(qkv, H, None, pos, cos, sin, norms[1], norms[2], norms[0])
        q, k, v = qkv.view(B, N, 3, H, d).permute(2, 0, 3, 1, 4).unbind(0)
        q, k = self.q_norm(q).to(v.dtype), self.k_norm(k).to(v.dtype)
        if turned:
            q, k = self.rope(q, xpos), self.rope(k, xpos)
        return q, k, v

    def forward(self, x: Tensor, attn_bias=None, xpos: Optional[Tensor] = None) -> Tensor:
        B, N, C = x.shape
        q, k, v = self._heads(self._linear(self.qkv, x), xpos, B, N, C // self.num_heads)
        drop = self.attn_drop                           # its own mode decides; an Identity has no p
        y = nn.functional.scaled_dot_product_attention(q, k, v, attn_mask=attn_bias, dropout_p=getattr(drop, "p", 0.0) if drop.training else 0.0)
        return self.proj_drop(self._linear(self.proj, y.transpose(1, 2).reshape(B, N, C)))
