"""B200 (sm_100a) implementation of Speed3R's dual-branch sparse global attention.

``SparseFlashAttentionRope`` is the drop-in module, ``BlockRope`` the block around it (8-bit projections for inference on request, or ``FusedMlp``
as its MLP), ``FlashAttentionRope`` the dense attention of the blocks in between,
``AdamW`` the optimiser of a training step; ``ops`` holds the reference-named operator functions; ``_lib`` binds the C-ABI library
declared in include/speed3r_b200.h.
"""
from .sparse_attention import RoPE2D, SparseFlashAttentionRope  # noqa: F401
from .ops import (flash_attn_topk_func, pool_tokens, sel_attn_merge,  # noqa: F401
                  topk_blocksparse_attention)
from .host_pipeline import HostPipeline  # noqa: F401
from .block import BlockRope, FusedMlp, forward_blocks  # noqa: F401
from .dense_attention import FlashAttentionRope  # noqa: F401
from .int8 import Int8Linear, Int8Tokens  # noqa: F401
from .optim import AdamW  # noqa: F401

__all__ = ["SparseFlashAttentionRope", "RoPE2D", "flash_attn_topk_func", "topk_blocksparse_attention",
           "pool_tokens", "sel_attn_merge", "HostPipeline", "BlockRope", "FusedMlp", "FlashAttentionRope", "forward_blocks", "Int8Linear", "Int8Tokens", "AdamW"]
