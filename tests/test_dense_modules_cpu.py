"""What the modules of the dense half of a block refuse, as far as no GPU is needed."""
import pytest
import torch
from torch import nn

from speed3r_b200 import BlockRope, FlashAttentionRope, FusedMlp


def test_dense_attention_has_no_8_bit_form():
    b = BlockRope(64, 1, attn_class=FlashAttentionRope, ffn_layer=FusedMlp)
    kept = {n: p.clone() for n, p in b.state_dict().items()}
    with pytest.raises(RuntimeError, match="FlashAttentionRope has no 8-bit form"):
        b.quantize_int8()
    assert type(b.mlp.fc1) is type(b.attn.qkv) is nn.Linear and all(torch.equal(p, kept[n]) for n, p in b.state_dict().items())
