"""The transformer block around the sparse attention, drop-in for the reference's ``BlockRope``.

``BlockRope`` keeps the constructor keywords, sub-module names (``norm1``, ``attn``, ``ls1``, ``norm2``, ``mlp.fc1``, ``mlp.fc2``, ``ls2``) and
``forward(x, xpos=None)`` of pi3/models/layers/block.py:259-335, so that a checkpoint loads unchanged.  What stands between its
sub-layers - LayerScale, stochastic depth, residual and the next norm - is ``ops.residual_norm``, one pass with gradients; the MLP's
matrices stay PyTorch (cuBLAS) code with ``Mlp``, are ``ops.linear`` with ``FusedMlp``, or become 8-bit products for inference (``quantize_int8``).  ``forward_blocks`` runs a list of blocks and
takes the sum that ends a block and the norm that begins the next one in one pass as well.
"""
from __future__ import annotations

from typing import Callable, Optional, Sequence, Tuple, Type, Union

import torch
from torch import Tensor, nn

from . import ops
from .int8 import Int8Linear, Int8Tokens
from .sparse_attention import SparseFlashAttentionRope, _global_hooks, _watched


class LayerScale(nn.Module):
    def __init__(self, dim: int, init_values: float = 1e-5):
        super().__init__()
        self.gamma = nn.Parameter(init_values * torch.ones(dim))

    def forward(self, x: Tensor) -> Tensor:
        return x * self.gamma


class Mlp(nn.Module):
    def __init__(self, in_features: int, hidden_features: Optional[int] = None, out_features: Optional[int] = None,
                 act_layer: Callable[..., nn.Module] = nn.GELU, drop: float = 0.0, bias: bool = True):
        super().__init__()
        self.fc1 = nn.Linear(in_features, hidden_features or in_features, bias=bias)
        self.act = act_layer()
        self.fc2 = nn.Linear(hidden_features or in_features, out_features or in_features, bias=bias)
        self.drop = nn.Dropout(drop)

    def forward(self, x) -> Tensor:
        return self.drop(self.fc2(self.drop(self.act(self.fc1(x)))))


def product_type(x, *linears: nn.Module) -> Optional[torch.dtype]:
    """The type in which ``ops.linear`` computes these Linears on x as autocast, or else x, wants them; None where they are to be called instead:
    something else than plain Linears, hooks, other types or devices."""
    if not isinstance(x, Tensor) or not x.is_cuda or _global_hooks() or any(type(m) is not nn.Linear or _watched(m) for m in linears):
        return None
    autocast = torch.is_autocast_enabled("cuda")
    t = torch.get_autocast_dtype("cuda") if autocast else x.dtype
    params = [p for m in linears for p in m._parameters.values() if p is not None]
    if t not in (torch.bfloat16, torch.float16) or any(p.device != x.device for p in params):
        return None
    if autocast:
        return t if x.dtype in ops.NORM_TYPES and all(p.dtype in ops.NORM_TYPES for p in params) else None
    return t if all(p.dtype == t for p in params) else None


class FusedMlp(Mlp):
    """``Mlp`` whose matrices come with what follows them (``ops.linear``): the activation, and on request a LayerScale and the residual.  For
    ``BlockRope(ffn_layer=FusedMlp)``; parameters and results are ``Mlp``'s, but that nothing is rounded between a matrix and its activation.  Where
    the kernel does not reach - other types than bf16 and fp16, active dropout, hooks, an activation other than GELU and SiLU, a residual or scale
    that is broadcast or has 64 bits - modules are called one by one.  Under autocast the weights are cast on every call."""

    def _act(self) -> Optional[str]:
        m = self.act
        if _watched(m):
            return None
        if type(m) is nn.GELU:
            return "gelu" if m.approximate == "none" else "gelu_tanh"
        return "silu" if type(m) is nn.SiLU else None

    def _type(self, x) -> Optional[torch.dtype]:
        d = self.drop
        if self._act() is None or _watched(d) or not (type(d) is nn.Identity or (type(d) is nn.Dropout and not (d.p and d.training))):
            return None
        return product_type(x, self.fc1, self.fc2)

    def _sums(self, x: Tensor, residual: Optional[Tensor], scale: Optional[Tensor]) -> bool:
        """The second product takes this residual and this scale: no types beyond the kernel's, nothing that is broadcast."""
        N = self.fc2.out_features
        return all(v is None or (v.dtype in ops.NORM_TYPES and v.device == x.device and v.shape == shape)
                   for v, shape in ((residual, (*x.shape[:-1], N)), (scale, (N,))))

    def forward(self, x, residual: Optional[Tensor] = None, scale: Optional[Tensor] = None) -> Tensor:
        """``residual + mlp(x) * scale``, in the residual's type, or without one in the MLP's own"""
        t = self._type(x)
        if t is None or not self._sums(x, residual, scale):
            y = super().forward(x)
            kept = y.dtype if residual is None else residual.dtype
            y = y if scale is None else y * scale
            return (y if residual is None else residual + y).to(kept)
        of = lambda p: None if p is None else p.to(t)
        h = ops.linear(x.to(t), of(self.fc1.weight), self.fc1.bias, self._act())
        return ops.linear(h, of(self.fc2.weight), self.fc2.bias, None, residual, scale, t if residual is None else residual.dtype)


def _norm_args(m: nn.Module, dim: int) -> Optional[Tuple[str, tuple]]:
    """(kind, (weight, bias, eps)) of a norm that ``ops.residual_norm`` computes, None for any other module."""
    if _watched(m):
        return None
    if type(m) is nn.LayerNorm and tuple(m.normalized_shape) == (dim,):
        return "layer", (m.weight, m.bias, m.eps)
    if type(m) is nn.RMSNorm and tuple(m.normalized_shape) == (dim,) and m.eps is not None:      # without one it depends on a type
        return "rms", (m.weight, None, m.eps)
    return None


class BlockRope(nn.Module):
    def __init__(
        self,
        dim: int,
        num_heads: int,
        mlp_ratio: float = 4.0,
        qkv_bias: bool = False,
        proj_bias: bool = True,
        ffn_bias: bool = True,
        drop: float = 0.0,
        attn_drop: float = 0.0,
        init_values: Optional[float] = None,
        drop_path: float = 0.0,
        act_layer: Callable[..., nn.Module] = nn.GELU,
        norm_layer: Callable[..., nn.Module] = nn.LayerNorm,
        attn_class: Type[nn.Module] = SparseFlashAttentionRope,
        ffn_layer: Callable[..., nn.Module] = Mlp,
        qk_norm: bool = False,
        rope=None,
    ) -> None:
        super().__init__()
        self.norm1 = norm_layer(dim)
        self.attn = attn_class(dim, num_heads=num_heads, qkv_bias=qkv_bias, proj_bias=proj_bias, attn_drop=attn_drop, proj_drop=drop,
                               qk_norm=qk_norm, rope=rope)
        self.ls1 = LayerScale(dim, init_values) if init_values else nn.Identity()
        self.norm2 = norm_layer(dim)
        self.mlp = ffn_layer(in_features=dim, hidden_features=int(dim * mlp_ratio), act_layer=act_layer, drop=drop, bias=ffn_bias)
        self.ls2 = LayerScale(dim, init_values) if init_values else nn.Identity()
        self.drop_path = float(drop_path)
        if not 0.0 <= self.drop_path < 1.0:
            raise ValueError(f"drop_path {drop_path}")
        self.dim = dim

    @torch.no_grad()
    def quantize_int8(self) -> "BlockRope":
        """8-bit projections and MLP for inference, in place (parameters on the GPU).  The norms then hand over 8-bit tokens.  For an
        MLP of two Linears ``fc1`` and ``fc2`` and an attention with an 8-bit form (``SparseFlashAttentionRope``); any other ``ffn_layer`` or
        ``attn_class`` raises, and nothing is changed."""
        if not callable(getattr(self.attn, "quantize_int8", None)):
            raise RuntimeError(f"quantize_int8: {type(self.attn).__name__} has no 8-bit form")
        lins = [getattr(self.mlp, n, None) for n in ("fc1", "fc2")]
        if not all(isinstance(m, (nn.Linear, Int8Linear)) for m in lins):
            raise RuntimeError(f"quantize_int8: {type(self.mlp).__name__} is not an MLP of two Linears fc1 and fc2")
        narrow = [m if type(m) is Int8Linear else Int8Linear.of(m) for m in lins]
        self.attn.quantize_int8()
        self.mlp.fc1, self.mlp.fc2 = narrow
        return self

    # ---- pieces ----------------------------------------------------------------------------------------------------------
    def _gate(self, x: Tensor) -> Optional[Tensor]:
        """Stochastic depth: a factor per sample, 0 or 1 / keep."""
        if not (self.training and self.drop_path):
            return None
        keep = 1.0 - self.drop_path
        return torch.empty((x.shape[0],) + (1,) * (x.dim() - 1), dtype=torch.float32, device=x.device).bernoulli_(keep).div_(keep)

    def _scale(self, m: nn.Module) -> Optional[Tensor]:
        return m.gamma if type(m) is LayerScale else None

    def _fuses(self) -> bool:
        """Norms and LayerScales are what they look like and nobody watches them."""
        return (_norm_args(self.norm1, self.dim) is not None and _norm_args(self.norm2, self.dim) is not None and not _global_hooks() and
                all(type(m) is nn.Identity or (type(m) is LayerScale and tuple(m.gamma.shape) == (self.dim,)) for m in (self.ls1, self.ls2)) and
                not any(_watched(m) for m in (self.ls1, self.ls2)))

    def _fits(self, x: Tensor) -> bool:
        """``ops.residual_norm`` has a kernel for this input: not on the CPU, of its types, no wider than it reaches."""
        params = (p for m in (self.norm1, self.norm2, self.ls1, self.ls2) for p in m._parameters.values() if p is not None)
        return (x.device.type != "cpu" and x.dtype in ops.NORM_TYPES and 1 <= x.shape[-1] <= ops.NORM_MAX_CHANNELS and
                all(p.dtype in ops.NORM_TYPES for p in params))

    def _residual(self, x: Tensor) -> Tensor:
        """x in the type that the sum with a scaled branch has."""
        kept = x.dtype
        for m in (self.ls1, self.ls2):
            if type(m) is LayerScale:
                kept = torch.promote_types(kept, m.gamma.dtype)
        return x.to(kept)

    @staticmethod
    def _narrow(x: Tensor) -> torch.dtype:
        """What the matrices are given."""
        return torch.get_autocast_dtype("cuda") if torch.is_autocast_enabled("cuda") else x.dtype

    @staticmethod
    def _sum_and_norm(x: Tensor, y: Optional[Tensor], norm: Optional[nn.Module], scale, gate, int8: bool):
        """(x + scale * gate * y, its norm)"""
        kind, args = _norm_args(norm, x.shape[-1]) if norm is not None else ("layer", None)
        if int8 and args is not None:
            r, q, s = ops.residual_norm_int8(x, y, args, scale, gate, kind=kind)
            return r, Int8Tokens(q, s)
        return ops.residual_norm(x, y, args, scale, gate, kind=kind, out_dtype=BlockRope._narrow(x))

    def _run(self, x: Tensor, h: Union[Tensor, Int8Tokens], xpos, next_norm: Optional[nn.Module], next_int8: bool):
        a = self.attn(h, xpos=xpos)
        x, h = self._sum_and_norm(x, a, self.norm2, self._scale(self.ls1), self._gate(x), self._mlp_takes_int8())
        if next_norm is None and type(self.mlp) is FusedMlp and not _watched(self.mlp) and not (self.training and self.drop_path) and self.mlp._type(h) is not None:
            return self.mlp(h, residual=x, scale=self._scale(self.ls2)), None            # nothing comes behind the sum: it leaves with the product
        return self._sum_and_norm(x, self.mlp(h), next_norm, self._scale(self.ls2), self._gate(x), next_int8)

    def _mlp_takes_int8(self) -> bool:
        """8-bit tokens are for the MLP whose first step is that Linear; another module is given activations."""
        return type(self.mlp) in (Mlp, FusedMlp) and type(self.mlp.fc1) is Int8Linear

    def _takes_int8(self) -> bool:
        return type(self.attn).forward is SparseFlashAttentionRope.forward and type(self.attn.qkv) is Int8Linear

    def forward(self, x: Tensor, xpos: Optional[Tensor] = None) -> Tensor:
        if not (self._fuses() and self._fits(x)):
            drop = lambda y: y if (g := self._gate(y)) is None else y * g.to(y.dtype)      # the branch keeps its type
            x = x + drop(self.ls1(self.attn(self.norm1(x), xpos=xpos)))
            return x + drop(self.ls2(self.mlp(self.norm2(x))))
        x = self._residual(x)
        _, h = self._sum_and_norm(x, None, self.norm1, None, None, self._takes_int8())
        return self._run(x, h, xpos, None, False)[0]


def forward_blocks(blocks: Sequence[BlockRope], x: Tensor, xpos: Optional[Tensor] = None) -> Tensor:
    """``for block in blocks: x = block(x, xpos)``, with the sum at the end of a block and the first norm of the next one in one pass."""
    blocks = list(blocks)
    if not all(type(b) is BlockRope and not _watched(b) and b._fuses() and b._fits(x) for b in blocks):
        for b in blocks:
            x = b(x, xpos=xpos)
        return x
    h = None
    for i, b in enumerate(blocks):
        wide = b._residual(x)
        if h is None or wide.dtype != x.dtype:
            _, h = b._sum_and_norm(wide, None, b.norm1, None, None, b._takes_int8())
        after = blocks[i + 1] if i + 1 < len(blocks) else None
        x, h = b._run(wide, h, xpos, after.norm1 if after is not None else None, after is not None and after._takes_int8())
    return x
