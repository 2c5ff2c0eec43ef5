"""Inference with 8-bit projections: weights as integers with a scale per output channel, activations per token."""
from __future__ import annotations

from typing import NamedTuple, Optional, Tuple, Union

import torch
from torch import Tensor, nn

from . import ops


class Int8Tokens(NamedTuple):
    """Activations ``q * scale`` in 8 bits, as ``ops.quantize_tokens`` and ``ops.residual_norm_int8`` make them."""
    q: Tensor
    scale: Tensor

    @property
    def shape(self):
        return self.q.shape

    requires_grad = False


class Int8Linear(nn.Module):
    """A Linear of 8-bit integers, without gradients: ``weight [N, K]`` int8, ``weight_scale [N]``, ``bias [N]`` fp32 or None.
    Takes activations (which it makes 8-bit tokens of) or ``Int8Tokens``; the result has ``out_dtype``."""

    def __init__(self, weight: Tensor, weight_scale: Tensor, bias: Optional[Tensor], out_dtype: torch.dtype = torch.bfloat16):
        super().__init__()
        self.register_buffer("weight", weight)
        self.register_buffer("weight_scale", weight_scale)
        self.register_buffer("bias", bias)
        self.out_features, self.in_features = weight.shape
        self.out_dtype = out_dtype

    @classmethod
    @torch.no_grad()
    def of(cls, *linears: nn.Linear, out_dtype: torch.dtype = torch.bfloat16) -> "Int8Linear":
        """The 8-bit form of a Linear on the GPU, or of several that read the same input, their outputs side by side."""
        for m in linears:
            if not isinstance(m, nn.Linear) or type(m).forward is not nn.Linear.forward or "forward" in m.__dict__:
                raise RuntimeError(f"Int8Linear.of: {type(m).__name__} computes something else than a Linear")
            if m._forward_hooks or m._forward_pre_hooks:              # they may change what goes in and out, or make the weight
                raise RuntimeError("Int8Linear.of: this Linear has hooks, which its 8-bit form would lose: remove them first")
        biases = [m.bias for m in linears]
        if any(b is None for b in biases) and any(b is not None for b in biases):
            biases = [b if b is not None else torch.zeros(m.out_features, device=m.weight.device) for b, m in zip(biases, linears)]
        q, scale = ops.quantize_tokens(torch.cat([m.weight.detach().float() for m in linears]))
        return cls(q, scale, None if biases[0] is None else torch.cat([b.detach().float() for b in biases]), out_dtype)

    def _apply(self, fn, recurse: bool = True):
        """Moves as any module; scales and bias stay fp32, which ``ops.int8_linear`` takes, through ``.bfloat16()`` and the like."""
        kept = {n: b for n, b in self._buffers.items() if n in ("weight_scale", "bias") and b is not None}
        super()._apply(fn, recurse)
        for n, b in kept.items():
            if self._buffers[n].dtype != b.dtype:
                self._buffers[n] = b.to(self._buffers[n].device)
        return self

    def forward(self, x: Union[Tensor, Int8Tokens]) -> Tensor:
        if not isinstance(x, Int8Tokens):
            x = Int8Tokens(*ops.quantize_tokens(x))
        return ops.int8_linear(x.q, x.scale, self.weight, self.weight_scale, self.bias, self.out_dtype)

    def extra_repr(self) -> str:
        return f"in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}, out_dtype={self.out_dtype}"


def tokens_of(x: Union[Tensor, Int8Tokens]) -> Int8Tokens:
    return x if isinstance(x, Int8Tokens) else Int8Tokens(*ops.quantize_tokens(x))
