"""The block, its 8-bit form and the optimiser as a program uses them, against PyTorch's own modules and optimiser; captured calls."""
import copy
import math

import pytest
import torch
from torch import nn

import speed3r_b200
from speed3r_b200 import AdamW, BlockRope, Int8Linear, Int8Tokens, forward_blocks, ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DIM, HEADS = 256, 4


def positions(B, T):
    tok = torch.arange(T, device=DEV) % 256
    return torch.stack((tok // 16, tok % 16), -1)[None].expand(B, -1, -1).contiguous()


def block(seed=0, **kw):
    torch.manual_seed(seed)
    b = BlockRope(DIM, HEADS, qkv_bias=True, qk_norm=True, rope=speed3r_b200.RoPE2D(100.0), **{"init_values": 0.3, **kw})
    with torch.no_grad():
        for name, p in b.named_parameters():
            if p.dim() == 2:
                p.normal_(0.0, 0.05)
            elif "norm" in name or "gamma" in name:
                p.add_(0.1 * torch.randn_like(p))
    return b.to(DEV)


def plain(b):
    """The same block with every module called by itself."""
    b._fuses = lambda: False
    return b


def near(got, want, share):
    """2-norm of the difference as a share of the result's."""
    off = (got.double() - want.double()).norm() / want.double().norm()
    assert off <= share, f"{off.item():.3g} > {share}"


# T = 512: 32 compressed keys, all of them selected, so that no rounding decides about a table.
@pytest.mark.parametrize("kw", [{}, dict(init_values=None), dict(norm_layer=lambda d: nn.RMSNorm(d, eps=1e-6)), dict(drop_path=0.4), dict(norm_layer=lambda d: nn.LayerNorm(d, bias=False))])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_block_and_its_gradients(kw, dtype):
    a, b = block(1, **kw), plain(block(1, **kw))
    B, T = 3, 512
    x = torch.randn(B, T, DIM, device=DEV).to(dtype)
    dy = torch.randn(B, T, DIM, device=DEV)
    got = []
    for m in (a, b):
        torch.manual_seed(7)
        xi = x.clone().requires_grad_(True)
        with torch.autocast("cuda", dtype=torch.bfloat16):
            y = m(xi, xpos=positions(B, T))
        y.float().backward(dy)
        got.append((y, xi.grad, dict(m.named_parameters())))
    (y, dx, p), (y2, dx2, p2) = got
    assert y.dtype == y2.dtype and dx.dtype == dx2.dtype
    # Both round branches, activations and their gradients to bf16 (2^-9 rms each) at the same places; the fused block does not round
    # the LayerScale's product in between.  A chain of about ten such roundings: 10 x 2^-9 = 2 %.
    near(y, y2, 0.02)
    near(dx, dx2, 0.02)
    for n in p:
        near(p[n].grad, p2[n].grad, 0.03 if p[n].dim() == 2 else 0.04)


def test_blocks_one_after_the_other():
    blocks = [block(i) for i in range(3)]
    x = torch.randn(2, 768, DIM, device=DEV)
    for context in (torch.no_grad(), torch.enable_grad()):
        with context, torch.autocast("cuda", dtype=torch.bfloat16):
            y = forward_blocks(blocks, x, positions(2, 768))
            z = x
            for b in blocks:
                z = b(z, positions(2, 768))
            assert torch.equal(y, z)
    watched = copy.deepcopy(blocks)
    seen = []
    watched[1].norm2.register_forward_hook(lambda m, i, o: seen.append(o.shape))
    with torch.no_grad(), torch.autocast("cuda", dtype=torch.bfloat16):
        near(forward_blocks(watched, x, positions(2, 768)), y, 0.02)
    assert len(seen) == 1


def test_block_in_bf16_without_autocast():
    a = block(2).bfloat16().eval()
    x = torch.randn(1, 512, DIM, device=DEV).bfloat16()
    with torch.no_grad():
        y, z = a(x, positions(1, 512)), plain(copy.deepcopy(a))(x, positions(1, 512))
    assert y.dtype == torch.bfloat16
    near(y, z, 0.02)


def test_int8_linear_module():
    torch.manual_seed(3)
    lins = [nn.Linear(200, n, bias=b).to(DEV) for n, b in ((72, True), (40, False))]
    m = Int8Linear.of(*lins)
    assert m.weight.shape == (112, 200) and m.weight.dtype == torch.int8
    x = torch.randn(3, 50, 200, device=DEV).bfloat16()
    y = m(x)
    q, s = ops.quantize_tokens(x)
    assert torch.equal(y, m(Int8Tokens(q, s))) and y.shape == (3, 50, 112) and y.dtype == torch.bfloat16
    want = torch.cat([nn.functional.linear(x.float(), l.weight, l.bias) for l in lins], -1)
    # two operands rounded to 8 bits, each by a step of max / 127 over sqrt(12): for a row of 200 normal values (largest about 3) 0.7 %
    near(y, want, 0.02)
    again = Int8Linear(torch.zeros_like(m.weight), torch.zeros_like(m.weight_scale), torch.zeros_like(m.bias))
    again.load_state_dict(m.state_dict())
    assert torch.equal(again(x), y)


def test_block_in_8_bits():
    a = block(4).eval()
    x = torch.randn(2, 512, DIM, device=DEV)
    with torch.no_grad(), torch.autocast("cuda", dtype=torch.bfloat16):
        want = a(x, positions(2, 512))
        q = copy.deepcopy(a).quantize_int8()
        got = q(x, positions(2, 512))
        # Branches of 0.3 LayerScales: each of four products in a row adds about 1 % of noise, the residual none.
        near(got - x, want - x, 0.06)
        h = ops.residual_norm(x, None, (a.norm1.weight, a.norm1.bias, a.norm1.eps), out_dtype=torch.bfloat16)[1]
        near(q.attn(h, xpos=positions(2, 512)), a.attn(h, xpos=positions(2, 512)), 0.06)
        two = [q, copy.deepcopy(block(5)).eval().quantize_int8()]
        assert torch.equal(forward_blocks(two, x, positions(2, 512)), two[1](two[0](x, positions(2, 512)), positions(2, 512)))
    with pytest.raises(RuntimeError, match="forward-only"):
        q(x.requires_grad_(True), positions(2, 512))


# ---- optimiser -------------------------------------------------------------------------------------------------------------
def nets(seed=0):
    torch.manual_seed(seed)
    m = nn.Sequential(nn.Linear(70, 333), nn.GELU(), nn.LayerNorm(333), nn.Linear(333, 1041), nn.GELU(), nn.Linear(1041, 5)).to(DEV)
    return m, copy.deepcopy(m)


def run(m, opt, clip, steps, skip=None):
    torch.manual_seed(1)
    for i in range(steps):
        opt.zero_grad(set_to_none=True)
        (m(torch.randn(64, 70, device=DEV)) ** 2).mean().backward()
        if skip and i in skip:
            for p in skip[i](m):
                p.grad = None
        if clip and isinstance(opt, torch.optim.AdamW):
            nn.utils.clip_grad_norm_(m.parameters(), clip)
        opt.step()


@pytest.mark.parametrize("clip", [None, 0.05])
def test_adamw_against_pytorch(clip):
    a, b = nets()
    groups = lambda m: [dict(params=[p for p in m.parameters() if p.dim() > 1], weight_decay=0.1), dict(params=[p for p in m.parameters() if p.dim() == 1], lr=3e-3, weight_decay=0.0)]
    # some parameters have no gradient at times, and the last layer none at first
    skip = {0: lambda m: m[5].parameters(), 1: lambda m: m[5].parameters(), 3: lambda m: m[0].parameters(), 4: lambda m: list(m.parameters())[1:4]}
    run(a, AdamW(groups(a), lr=1e-3, betas=(0.8, 0.95), max_norm=clip), clip, 8, skip)
    run(b, torch.optim.AdamW(groups(b), lr=1e-3, betas=(0.8, 0.95)), clip, 8, skip)
    for p, q in zip(a.parameters(), b.parameters()):
        # eight steps of at most lr each, off by a few 2^-23 of a step, and what that does to later gradients
        assert ((p - q).abs() <= 1e-6 * q.abs() + 1e-5 * 3e-3 * 8).all()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_adamw_continues_from_a_state_dict(bits, dtype, tmp_path):
    a, b = (m.to(dtype) for m in nets(2))
    make = lambda m: AdamW(m.parameters(), lr=1e-3, state_bits=bits, max_norm=1.0, min_8bit_size=1000)
    def go(m, opt, steps, seed):
        torch.manual_seed(seed)
        for _ in range(steps):
            opt.zero_grad()
            (m(torch.randn(64, 70, device=DEV, dtype=dtype)) ** 2).float().mean().backward()
            opt.step()
    oa = make(a)
    go(a, oa, 3, 1)
    torch.save(dict(m=a.state_dict(), o=oa.state_dict()), tmp_path / "s.pt")
    go(a, oa, 3, 2)
    saved = torch.load(tmp_path / "s.pt")
    b.load_state_dict(saved["m"])
    ob = make(b)
    ob.load_state_dict(saved["o"])
    go(b, ob, 3, 2)
    assert all(torch.equal(p, q) for p, q in zip(a.parameters(), b.parameters()))
    kinds = {s["exp_avg"].dtype for s in ob.state.values()}
    assert kinds == ({torch.float32, torch.uint8} if bits == 8 else {torch.float32})
    assert len({id(s["step"]) for s in ob.state.values()}) == 1


def test_adamw_refuses():
    p = nn.Parameter(torch.zeros(4, device=DEV))
    for kw in (dict(lr=-1.0), dict(betas=(1.0, 0.9)), dict(eps=-1.0), dict(weight_decay=-1.0), dict(max_norm=0.0), dict(state_bits=16)):
        with pytest.raises(ValueError):
            AdamW([p], **kw)
    x = torch.zeros(8, device=DEV)
    step = torch.zeros((), dtype=torch.int64, device=DEV)
    with pytest.raises(RuntimeError, match="listed twice"):
        ops.adamw_step([x, x], [x, x], [x.clone(), x.clone()], [x.clone(), x.clone()], step)
    for kw, text in ((dict(params=[torch.zeros(4, 4, device=DEV).t()[:2]]), "contiguous"), (dict(grads=[torch.zeros(7, device=DEV)]), "gradient"), (dict(exp_avg=[torch.zeros(8, device=DEV).bfloat16()]), "state"),
                     (dict(step=torch.zeros((), device=DEV)), "step"), (dict(scales=[torch.zeros(2, 1, device=DEV, dtype=torch.uint8)]), "state"), (dict(exp_avg_sq=[]), "states"),
                     (dict(params=[torch.zeros(8, device=DEV, dtype=torch.float64)]), "fp32, bf16 or fp16")):
        args = dict(params=[x], grads=[x.clone()], exp_avg=[x.clone()], exp_avg_sq=[x.clone()], step=step)
        args.update(kw)
        if "params" in kw and kw["params"][0].dim() == 2:
            args["grads"] = [torch.zeros(2, 4, device=DEV)]
        with pytest.raises(RuntimeError, match=text):
            ops.adamw_step(**args)
    assert int(step) == 0


# ---- together --------------------------------------------------------------------------------------------------------------
def test_training_steps_of_a_block():
    """Block, clipping and update as a training loop runs them, against the same block and optimiser of PyTorch's parts."""
    a, b = block(6), plain(block(6))
    x, dy = torch.randn(2, 512, DIM, device=DEV), torch.randn(2, 512, DIM, device=DEV)
    start = {n: p.detach().clone() for n, p in a.named_parameters()}
    for m in (a, b):
        opt = AdamW(m.parameters(), lr=1e-3, max_norm=1.0) if m is a else torch.optim.AdamW(m.parameters(), lr=1e-3)
        for _ in range(3):
            opt.zero_grad()
            with torch.autocast("cuda", dtype=torch.bfloat16):
                y = m(x, xpos=positions(2, 512))
            y.backward(dy)
            if m is b:
                nn.utils.clip_grad_norm_(m.parameters(), 1.0)
            opt.step()
    # Adam's steps are near lr in size whatever the gradient, and of either sign where it is near zero: matrices are compared as a whole
    moved = lambda m, n: dict(m.named_parameters())[n].detach() - start[n]
    for n in start:
        if start[n].dim() == 2 and "gate" not in n:
            near(moved(a, n), moved(b, n), 0.15)


@pytest.mark.parametrize("seed", [None, 5])
def test_captured_training_step(seed):
    """Norm, its gradients, clipping and update in one graph, replayed: the bits of eager steps."""
    def make():
        torch.manual_seed(8)
        w, b, s = (nn.Parameter(torch.randn(1024, device=DEV)) for _ in range(3))
        big = nn.Parameter(torch.randn(1024, 1024, device=DEV))
        opt = AdamW([w, b, s, big], lr=torch.tensor(1e-2, device=DEV), state_bits=8, max_norm=1.0, seed=seed)
        return (w, b, s, big), opt

    x, y = torch.randn(4, 700, 1024, device=DEV), torch.randn(4, 700, 1024, device=DEV).bfloat16()

    def one(params, opt):
        w, b, s, big = params
        opt.zero_grad()
        r, h = ops.residual_norm(x, y, (w, b, 1e-5), s, out_dtype=torch.bfloat16)
        ((r * 0.1).sum() + (h.float() * 0.01).square().sum() + (big * 0.01).square().sum()).backward()
        opt.step()

    def rounds(params, opt, graph):
        for _ in range(3):
            one(params, opt)
        if graph:
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                one(params, opt)
            torch.cuda.current_stream().wait_stream(side)
            for p in params:
                p.grad = None
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                one(params, opt)
            for i in range(4):
                if i == 2:
                    opt.param_groups[0]["lr"].fill_(1e-3)
                g.replay()
        else:
            for i in range(5):
                if i == 3:
                    opt.param_groups[0]["lr"].fill_(1e-3)
                one(params, opt)
        torch.cuda.synchronize()
        return [p.detach().clone() for p in params] + [opt.state[p]["step"].clone() for p in params]

    assert all(torch.equal(p, q) for p, q in zip(rounds(*make(), False), rounds(*make(), True)))


def test_two_captured_products_share_nothing():
    q, w = (torch.randint(-127, 128, s, device=DEV, dtype=torch.int8) for s in ((500, 1024), (1000, 1024)))
    s, ws = torch.rand(500, device=DEV), torch.rand(1000, device=DEV)
    x = torch.randn(500, 1024, device=DEV).bfloat16()
    want, want_x = ops.int8_linear(q, s, w, ws), ops.int8_linear(*ops.quantize_tokens(x), w, ws)
    graphs = []
    for part in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = ops.int8_linear(q, s, w, ws) if part == 0 else ops.int8_linear(*ops.quantize_tokens(x), w, ws)
        graphs.append((g, out))
    for _ in range(3):
        for g, _ in reversed(graphs):
            g.replay()
    # side by side, on streams of their own
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for st, (g, _) in zip(streams, graphs):
        with torch.cuda.stream(st):
            g.replay()
    torch.cuda.synchronize()
    assert torch.equal(graphs[0][1], want) and torch.equal(graphs[1][1], want_x)


def test_other_streams():
    x, y = torch.randn(3, 1041, 1024, device=DEV), torch.randn(3, 1041, 1024, device=DEV).bfloat16()
    w = torch.randn(1024, device=DEV)
    r, h = ops.residual_norm(x, y, (w, None, 1e-5), w, kind="rms")
    q, s = ops.quantize_tokens(h)
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        r2, h2 = ops.residual_norm(x, y, (w, None, 1e-5), w, kind="rms")
        q2, s2 = ops.quantize_tokens(h2)
        n2 = ops.grad_norm([h2, x])
    st.synchronize()
    assert torch.equal(r, r2) and torch.equal(h, h2) and torch.equal(q, q2) and torch.equal(s, s2)
    assert torch.equal(n2, ops.grad_norm([h, x]))


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_other_device_than_the_current_one():
    with torch.cuda.device(0):
        x = torch.randn(5, 256, device="cuda:1")
        w = torch.ones(256, device="cuda:1")
        r, h = ops.residual_norm(x, x, (w, w, 1e-5))
        q, s = ops.quantize_tokens(h)
        assert ops.int8_linear(q, s, q, s).device == x.device and ops.grad_norm([x]).device == x.device
        with pytest.raises(RuntimeError):
            ops.residual_norm(x, x.to("cuda:0"), (w, w, 1e-5))
