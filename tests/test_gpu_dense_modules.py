"""FusedMlp and FlashAttentionRope where their modules are replaced, watched or given what the kernels do not take."""
import itertools

import pytest
import torch
from torch import nn

from speed3r_b200 import FusedMlp, _lib, forward_blocks
from test_gpu_block import DEV, DIM, block, near, positions
from test_gpu_dense_block import attention, launched, mlps

pytestmark = pytest.mark.gpu
BF16, F16, FP32, FP64 = torch.bfloat16, torch.float16, torch.float32, torch.float64


@pytest.fixture(autouse=True)
def no_status():
    _lib.device_status()
    yield
    assert _lib.device_status() == 0


def fused(f):
    return sum("linear_kernel" in n or "linear_few" in n for n in launched(f)) == 2


@pytest.mark.parametrize("residual, scale", list(itertools.product((None, BF16, F16, FP32, FP64), repeat=2)))
def test_the_type_of_the_sum(residual, scale):
    """The residual's, or the MLP's own, whichever way the modules are called."""
    a, _ = mlps(dtype=BF16)
    torch.manual_seed(3)
    x = torch.randn(2, 9, DIM, device=DEV).to(BF16)
    r = None if residual is None else torch.randn(2, 9, DIM, device=DEV).to(residual)
    s = None if scale is None else torch.randn(DIM, device=DEV).to(scale)
    with torch.no_grad():
        assert fused(lambda: a(x, r, s)) == (FP64 not in (residual, scale))
        y = a(x, r, s)
        hook = a.fc1.register_forward_hook(lambda m, i, o: None)
        z = a(x, r, s)
        hook.remove()
    assert y.dtype == z.dtype == (residual or BF16)
    near(y, z, 0.02)                                             # four roundings of 2^-9 in the modules, half as many in the products


def test_a_sum_that_is_broadcast():
    a, b = mlps(dtype=BF16)
    x = torch.randn(2, 9, DIM, device=DEV).to(BF16)
    row, s = torch.randn(DIM, device=DEV), torch.randn(DIM, device=DEV)
    with torch.no_grad():
        want = b(x)
        for r, f in ((row, s), (row[None, None], None), (None, s[0]), (None, s[None, None]), (torch.randn(3, 2, 9, DIM, device=DEV), s), (torch.randn(2, 1, DIM, device=DEV), s[:1])):
            y = a(x, r, f)
            z = want.float() * (1 if f is None else f) + (0 if r is None else r)
            assert y.shape == z.shape and y.dtype == (BF16 if r is None else FP32)
            near(y, z, 0.01)


def test_a_dropout_that_was_replaced():
    class Half(nn.Module):
        def forward(self, x):
            return x * 0.5

    x = torch.randn(3, DIM, device=DEV).to(BF16)
    for drop, takes in ((nn.Identity(), True), (Half(), False), (nn.AlphaDropout(0.0), False), (nn.Dropout(0.5).eval(), True)):
        a, b = mlps(dtype=BF16)
        a.drop = b.drop = drop
        with torch.no_grad():
            assert fused(lambda: a(x)) == takes
            near(a(x), b(x), 0.01)


def test_attention_goes_by_its_own_dropout():
    m = attention(1, dtype=BF16, rope=None, attn_drop=0.5).train()
    x = torch.randn(2, 50, DIM, device=DEV).to(BF16)
    assert not torch.equal(m(x), m(x))
    m.attn_drop.eval()
    y = m(x)
    assert torch.equal(y, m(x))
    m.attn_drop = nn.Identity()
    assert torch.equal(y, m.train()(x)) and torch.equal(y, m.eval()(x))


@pytest.mark.parametrize("kw", [{}, dict(qk_norm=False), dict(rope=None), dict(norm_layer=lambda d: nn.RMSNorm(d, eps=1e-6)), dict(dim=4 * 48), dict(dim=4 * 128)])
def test_gradient_of_the_projections_bias(kw):
    """Of q, k and v: the sum over tokens of the projection's own gradient, in 32 bits; and for q and v the modules' (for k the sum nearly cancels
    where rotation is slow: what is added to all keys alike changes no softmax)."""
    C = kw.get("dim", DIM)
    torch.manual_seed(2)
    x, dy = torch.randn(3, 200, C, device=DEV), torch.randn(3, 200, C, device=DEV)
    grads = []
    for plain in (False, True):
        m, kept = attention(1, plain=plain, **kw), []
        heads = m._heads

        def watched(qkv, *args):
            qkv.retain_grad()
            kept.append(qkv)
            return heads(qkv, *args)

        m._heads = watched
        with torch.autocast("cuda", dtype=BF16):
            y = m(x, xpos=positions(3, 200))
        y.float().backward(dy)
        grads.append(m.qkv.bias.grad)
        if not plain:
            d = kept[0].grad.double().flatten(0, 1)
            # 600 terms, each addition off by at most 2^-24 of the magnitudes so far
            assert ((grads[0].double() - d.sum(0)).abs() <= 600 * 2.0 ** -24 * d.abs().sum(0)).all() and (grads[0] != 0).any()
    for i in (0, 2):
        near(grads[0].view(3, C)[i], grads[1].view(3, C)[i], 0.04)           # as every other parameter's: about sixteen roundings of 2^-9


def test_8_bit_blocks_with_either_mlp_are_one():
    """Their norms hand over 8-bit tokens to both: the same kernels, the same bits."""
    x, pos = torch.randn(2, 512, DIM, device=DEV), positions(2, 512)
    kinds = [[block(i, **kw).eval().quantize_int8() for i in range(2)] for kw in ({}, dict(ffn_layer=FusedMlp))]
    with torch.no_grad(), torch.autocast("cuda", dtype=torch.bfloat16):
        for blocks in kinds:
            forward_blocks(blocks, x, pos)                       # what is set up once has been
        names = [launched(lambda: forward_blocks(blocks, x, pos)) for blocks in kinds]
        assert names[0] == names[1] and any("int8" in n for n in names[0])
        assert torch.equal(*(forward_blocks(blocks, x, pos) for blocks in kinds))
