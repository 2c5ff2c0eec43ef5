"""FusedMlp and the dense attention module as a program uses them, against the modules that they stand for."""
import pytest
import torch
from torch import nn

import speed3r_b200
from speed3r_b200 import BlockRope, FlashAttentionRope, FusedMlp, forward_blocks
from speed3r_b200.block import Mlp
from test_gpu_block import DEV, DIM, HEADS, block, near, positions

pytestmark = pytest.mark.gpu


def launched(f):
    """Names of the kernels that f() launches."""
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CUDA]) as p:
        f()
        torch.cuda.synchronize()
    return [e.name for e in p.events() if e.device_type == torch.autograd.DeviceType.CUDA]


def mlps(act=nn.GELU, seed=0, dtype=torch.float32, **kw):
    torch.manual_seed(seed)
    a, b = FusedMlp(DIM, 4 * DIM, act_layer=act, **kw).to(DEV, dtype), Mlp(DIM, 4 * DIM, act_layer=act, **kw).to(DEV, dtype)
    b.load_state_dict(a.state_dict())
    return a, b


@pytest.mark.parametrize("act", [nn.GELU, lambda: nn.GELU("tanh"), nn.SiLU])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_mlp_and_its_gradients(act, dtype):
    a, b = mlps(act, dtype=dtype)
    x, dy = torch.randn(2, 70, DIM, device=DEV).to(dtype), torch.randn(2, 70, DIM, device=DEV)
    results = []
    for m in (a, b):
        xi = x.clone().requires_grad_(True)
        with torch.autocast("cuda", dtype=torch.bfloat16, enabled=dtype == torch.float32):
            y = m(xi)
        y.float().backward(dy)
        results.append((y, xi.grad, {n: p.grad for n, p in m.named_parameters()}))
    (y, dx, p), (y2, dx2, p2) = results
    assert y.dtype == y2.dtype and dx.dtype == dx2.dtype
    # Mlp rounds in front of the activation as well: three roundings forward, twice as many back, 2^-9 at most each
    near(y, y2, 0.01)
    near(dx, dx2, 0.02)
    for n in p:
        assert p[n].dtype == p2[n].dtype
        near(p[n], p2[n], 0.02)


def test_mlp_of_other_kinds_calls_its_modules():
    x = torch.randn(3, DIM, device=DEV)
    a, b = mlps()
    assert torch.equal(a(x), b(x))                                          # fp32
    a, b = mlps(nn.ReLU, dtype=torch.bfloat16)
    assert torch.equal(a(x.bfloat16()), b(x.bfloat16()))                    # another activation
    a, b = mlps(dtype=torch.bfloat16)
    seen = []
    hook = a.fc1.register_forward_hook(lambda m, i, o: seen.append(1))
    assert torch.equal(a(x.bfloat16()), b(x.bfloat16())) and seen
    hook.remove()
    assert any("linear" in n and "s3r" in n for n in launched(lambda: a(x.bfloat16())))
    a, b = mlps(dtype=torch.bfloat16, drop=0.5)
    torch.manual_seed(1)
    y = a(x.bfloat16())
    torch.manual_seed(1)
    assert torch.equal(y, b(x.bfloat16()))
    a, b = mlps(dtype=torch.bfloat16)
    r, s = torch.randn(3, DIM, device=DEV), torch.randn(DIM, device=DEV)
    for m in (a, mlps(nn.ReLU, dtype=torch.bfloat16)[0]):
        y = m(x.bfloat16(), residual=r, scale=s)
        assert y.dtype == torch.float32
        near(y - r, m(x.bfloat16()).float() * s, 0.01)


@pytest.mark.parametrize("kw", [{}, dict(init_values=None), dict(drop_path=0.4)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_block_with_it(kw, dtype):
    """T = 512: 32 compressed keys, all selected."""
    a, b = block(1, ffn_layer=FusedMlp, **kw), block(1, **kw)
    x, dy = torch.randn(3, 512, DIM, device=DEV).to(dtype), torch.randn(3, 512, DIM, device=DEV)
    got = []
    for m in (a, b):
        torch.manual_seed(7)
        xi = x.clone().requires_grad_(True)
        with torch.autocast("cuda", dtype=torch.bfloat16):
            y = m(xi, xpos=positions(3, 512))
        y.float().backward(dy)
        got.append((y, xi.grad, dict(m.named_parameters())))
    (y, dx, p), (y2, dx2, p2) = got
    assert y.dtype == y2.dtype and dx.dtype == dx2.dtype
    near(y, y2, 0.02)                                                       # as between the block's other forms: about ten roundings to bf16
    near(dx, dx2, 0.02)
    for n in p:
        near(p[n].grad, p2[n].grad, 0.03 if p[n].dim() == 2 else 0.04)


def test_block_quantises_with_it():
    b = block(2, ffn_layer=FusedMlp).eval()
    x = torch.randn(1, 512, DIM, device=DEV)
    with torch.no_grad(), torch.autocast("cuda", dtype=torch.bfloat16):
        y = b(x, xpos=positions(1, 512))
        b.quantize_int8()
        near(b(x, xpos=positions(1, 512)), y, 0.03)


# ---- dense attention -------------------------------------------------------------------------------------------------------
def attention(seed=0, dim=DIM, heads=HEADS, plain=False, dtype=torch.float32, **kw):
    torch.manual_seed(seed)
    m = FlashAttentionRope(dim, heads, qkv_bias=True, **{"qk_norm": True, "rope": speed3r_b200.RoPE2D(100.0), **kw}).to(DEV, dtype)
    if plain:
        m._norms = lambda d: None                       # norms and rotary module one by one
        m._linear = lambda lin, x: lin(x)
    return m


@pytest.mark.parametrize("kw", [{}, dict(qk_norm=False), dict(rope=None), dict(norm_layer=lambda d: nn.RMSNorm(d, eps=1e-6)), dict(dim=4 * 48), dict(dim=4 * 128)])
def test_attention_and_its_gradients(kw):
    a, b = attention(1, **kw), attention(1, plain=True, **kw)
    C = kw.get("dim", DIM)
    x, dy = torch.randn(3, 200, C, device=DEV), torch.randn(3, 200, C, device=DEV)
    got = []
    for m in (a, b):
        xi = x.clone().requires_grad_(True)
        with torch.autocast("cuda", dtype=torch.bfloat16):
            y = m(xi, xpos=positions(3, 200))
        y.float().backward(dy)
        got.append((y, xi.grad, {n: p.grad for n, p in m.named_parameters()}))
    (y, dx, p), (y2, dx2, p2) = got
    assert y.dtype == y2.dtype == torch.bfloat16
    # the modules round after the norm and within the rotation as well; about eight roundings of 2^-9, twice that back
    near(y, y2, 0.02)
    near(dx, dx2, 0.03)
    for n in p:
        # What is added to all keys alike changes no softmax: the sum over keys j of dS_ij = P_ij (dP_ij - sum_k P_ik dP_ik) is 0.  Such gradients are
        # roundings and nothing else: the keys' part of qkv.bias without norms, k_norm.bias without a rotation.
        if n != "qkv.bias" and not (n == "k_norm.bias" and m.rope is None):
            near(p[n], p2[n], 0.04)


def test_attention_of_other_kinds_calls_its_modules():
    class Scaled(nn.LayerNorm):
        def forward(self, x):
            return super().forward(x) * 2

    x = torch.randn(2, 50, DIM, device=DEV).bfloat16()
    pos = positions(2, 50)
    a, b = attention(1, dtype=torch.bfloat16, norm_layer=Scaled), attention(1, plain=True, dtype=torch.bfloat16, norm_layer=Scaled)
    near(a(x, xpos=pos), b(x, xpos=pos), 0.01)
    a = attention(1, dtype=torch.bfloat16)
    y, seen = a(x, xpos=pos), []
    hook = a.q_norm.register_forward_hook(lambda m, i, o: seen.append(1))
    near(a(x, xpos=pos), y, 0.02)
    assert seen
    hook.remove()
    names = launched(lambda: a(x, xpos=pos))
    assert sum("norm_rope" in n for n in names) == 1 and sum("linear_kernel" in n for n in names) == 2
    full = attention(1)
    assert full(x.float(), xpos=pos).dtype == torch.float32                 # fp32 without autocast: PyTorch's products


def test_frame_and_global_blocks_in_a_row():
    """A frame block (dense attention inside views) in front of a global one, as the decoder has them, trained a step."""
    rope = speed3r_b200.RoPE2D(100.0)
    torch.manual_seed(0)
    kw = dict(qkv_bias=True, qk_norm=True, init_values=0.3, ffn_layer=FusedMlp, rope=rope)
    frame, whole = BlockRope(DIM, HEADS, attn_class=FlashAttentionRope, **kw).to(DEV), BlockRope(DIM, HEADS, **kw).to(DEV)
    x = torch.randn(2, 256, DIM, device=DEV, requires_grad=True)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = frame(x, xpos=positions(2, 256))
        y = whole(y.view(1, 512, DIM), xpos=positions(1, 512))
        z = forward_blocks([frame, frame], x, positions(2, 256))
    assert z.shape == x.shape
    y.square().mean().backward()
    assert torch.isfinite(x.grad).all() and all(torch.isfinite(p.grad).all() for m in (frame, whole) for p in m.parameters())
