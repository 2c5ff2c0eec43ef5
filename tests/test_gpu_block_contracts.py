"""What the operators around the attention promise beyond their formulas: tracing, random numbers, extreme arguments, kernels chosen by size."""
import math

import pytest
import torch

from speed3r_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U8 = torch.uint8


def compiled(f):
    ops._ops()
    torch._dynamo.reset()
    return torch.compile(f, backend="aot_eager", fullgraph=True)


def state(shapes, eight, seed=0, dtype=torch.float32):
    """Parameters, gradients, first and second moments, scales (None: 32 bits) and the step's number."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    rand = lambda s: torch.randn(s, device=DEV, generator=g)
    params, grads = ([rand(s).to(dtype) for s in shapes] for _ in range(2))
    first, second, scales = [], [], []
    for s, e in zip(shapes, eight):
        codes = lambda: torch.randint(0, 120, s, device=DEV, dtype=U8, generator=g)
        first.append(codes() if e else 0.1 * rand(s))
        second.append(codes() if e else rand(s) ** 2)
        scales.append(torch.randint(115, 125, (2, -(-math.prod(s) // 256)), device=DEV, dtype=U8, generator=g) if e else None)
    return params, grads, first, second, scales, torch.tensor(3, device=DEV)


# ---- tracing ---------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("eight", [(True, False, True), (False, False, False)])
def test_compiled_step_is_the_step(eight):
    shapes = [(300,), (17, 5), (1041,)]
    some = lambda: state(shapes, eight, seed=1)

    def f(params, grads, first, second, scales, step):
        # values of before and of after, which a tracer must not take for the same
        held = [t for t in first + second + scales if t is not None]
        before = [t + 1 for t in held]
        norm = ops.grad_norm(grads)
        ops.adamw_step(params, grads, first, second, step, lr=1e-2, grad_norm=norm, max_norm=1.0, scales=scales if any(eight) else None, seed=5)
        return before, [t + 1 for t in held], norm

    a, b = some(), some()
    want, got = f(*a), compiled(f)(*b)
    flat = lambda x: [t for y in x for t in (flat(y) if isinstance(y, (list, tuple)) else [y]) if t is not None]
    assert len(flat(want)) == len(flat(got)) and all(torch.equal(x, y) for x, y in zip(flat(want) + flat(a), flat(got) + flat(b)))


@pytest.mark.parametrize("post", [False, True])
def test_compiled_norms_are_the_norms(post):
    """Forward and backward, through the nodes that a tracer sees."""
    gen = torch.Generator(device=DEV).manual_seed(2)
    rand = lambda *s: torch.randn(*s, device=DEV, generator=gen)
    inputs = [rand(2, 33, 136), rand(2, 33, 136).bfloat16(), rand(136), rand(136), rand(136), rand(2, 33, 1), rand(136)]

    def f(x, y, w, b, scale, gate, pw):
        r, h = ops.residual_norm(x, y, (w, b, 1e-5), scale, gate, (pw, None, 1e-6) if post else None, "rms" if post else "layer", torch.bfloat16)
        return (r * 2).sum() + (h.float() ** 2).sum(), r, h

    results = []
    for call in (f, compiled(f)):
        leaves = [t.clone().requires_grad_(True) for t in inputs]
        loss, r, h = call(*leaves)
        loss.backward()
        results.append([r.detach(), h.detach()] + [t.grad for t in leaves[:6 + post]])
    assert all(torch.equal(a, b) for a, b in zip(*results)) and len(results[0]) == 8 + post


def test_compiled_8_bit_products_are_the_products():
    x, w = torch.randn(3, 7, 72, device=DEV).bfloat16(), torch.randn(40, 72, device=DEV)
    wq, ws = ops.quantize_tokens(w)
    bias, one = torch.randn(40, device=DEV), torch.ones(72, device=DEV)

    def f(x):
        r, q, s = ops.residual_norm_int8(x, x, (one, None, 1e-5))
        return r, ops.int8_linear(q, s, wq, ws, bias), ops.int8_linear(*ops.quantize_tokens(x), wq, ws, None, torch.float32)

    with torch.no_grad():
        assert all(torch.equal(a, b) for a, b in zip(f(x), compiled(f)(x)))


def test_operators_have_the_schemas_and_shapes_that_they_say():
    x, y, w = torch.randn(2, 3, 40, device=DEV), torch.randn(2, 3, 40, device=DEV).bfloat16(), torch.ones(40, device=DEV)
    check = lambda op, args: torch.library.opcheck(op, args, test_utils=("test_schema", "test_faketensor"))
    ns = ops._ops()
    args = (x, y, w, w, w, None, None, None)
    r, h, stats = ns.residual_norm_fwd(*args, True, False, 0, 1e-5, 0.0, torch.bfloat16, True)
    check(ns.residual_norm_fwd.default, (*args, True, False, 0, 1e-5, 0.0, torch.bfloat16, True))
    check(ns.residual_norm_int8.default, (*args, False, 0, 1e-5, 0.0))
    check(ns.residual_norm_bwd.default, (r, y, w, w, None, None, None, stats, x, h, torch.bfloat16, False, 0, 31, torch.float32))
    check(ns.quantize_rows.default, (x,))
    q, s = ops.quantize_tokens(x)
    check(ns.int8_product.default, (q, s, q.reshape(6, 40), s.reshape(6), None, torch.float16))
    check(ns.norm_of.default, ([x, y],))
    p, g, m, v, e, step = state([(300,), (7,)], (True, False))
    check(ns.adamw_update.default, (p, g, m, v, step, [e[0]], 1e-3, None, 0.9, 0.99, 1e-8, 0.1, None, 0.0, 3))
    check(ns.adamw_values.default, (m[:1], v[:1], e[:1], [torch.zeros(300, device=DEV)], [torch.zeros(300, device=DEV)]))


def test_what_is_written_counts_as_changed():
    """Autograd notices that a tensor which it has saved was written: every tensor that a call changes, and no other."""
    p, g, m, v, e, step = state([(300,), (1041,)], (True, False))
    norm = ops.grad_norm(g)
    changed, read = p + m + v + e[:1] + [step], g + [norm]
    versions = lambda ts: [t._version for t in ts]
    before, kept = versions(changed), versions(read)
    ops.adamw_step(p, g, m, v, step, grad_norm=norm, scales=e)
    assert all(b > a for a, b in zip(before, versions(changed))) and versions(read) == kept
    out = [torch.zeros(300, device=DEV)], [torch.zeros(300, device=DEV)]
    read = m + v + e[:1]
    before, kept = versions(out[0] + out[1]), versions(read)
    ops.adamw_state(m[:1], v[:1], e[:1], out=out)
    assert all(b > a for a, b in zip(before, versions(out[0] + out[1]))) and versions(read) == kept
    w = torch.ones((), device=DEV, requires_grad=True)
    y = (w * out[0][0]).sum()
    ops.adamw_state(m[:1], v[:1], e[:1], out=out)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    with torch.inference_mode():
        frozen = state([(300,)], (True,))
        ops.adamw_step(*frozen[:4], frozen[5], scales=frozen[4])


# ---- the block -------------------------------------------------------------------------------------------------------------
def block(dim=128, **kw):
    from speed3r_b200 import BlockRope
    torch.manual_seed(0)
    return BlockRope(dim, dim // 64, **kw).to(DEV)


def by_modules(b, x):
    """The block's formula, every module called by itself."""
    x = x + b.ls1(b.attn(b.norm1(x)))
    return x + b.ls2(b.mlp(b.norm2(x)))


def test_a_scale_of_another_formula_takes_part():
    from speed3r_b200.block import LayerScale

    class Exponential(LayerScale):
        def forward(self, x):
            return x * self.gamma.exp()

    b = block(init_values=0.1)
    b.ls1 = Exponential(128, 0.1).to(DEV)
    x = torch.randn(2, 512, 128, device=DEV)
    with torch.no_grad(), torch.autocast("cuda", dtype=torch.bfloat16):
        assert torch.equal(b(x), by_modules(b, x))


def test_block_with_another_feed_forward_layer():
    from test_block_contracts_cpu import Gated
    from speed3r_b200 import forward_blocks

    b = block(ffn_layer=Gated, init_values=0.1)
    x = torch.randn(2, 512, 128, device=DEV, requires_grad=True)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y, z = b(x), by_modules(b, x)
        assert torch.equal(forward_blocks([b], x), y)
    # branches and activations are rounded to bf16 at the same places but for the LayerScales' products: 2^-9 rms each, a chain of ten
    assert (y - z).norm() <= 0.02 * z.norm()
    (g,) = torch.autograd.grad(y.sum(), x)
    (h,) = torch.autograd.grad(z.sum(), x)
    assert (g - h).norm() <= 0.02 * h.norm()


def test_an_mlp_that_is_not_ours_is_given_activations_in_8_bits_too():
    from speed3r_b200 import Int8Linear, Int8Tokens
    from speed3r_b200.block import Mlp

    class Other(Mlp):
        def forward(self, x):
            assert not isinstance(x, Int8Tokens)
            return super().forward(x.float().clamp(-2, 2))

    b = block(ffn_layer=Other).eval()
    x = torch.randn(2, 512, 128, device=DEV)
    with torch.no_grad(), torch.autocast("cuda", dtype=torch.bfloat16):
        want = b(x)
        got = b.quantize_int8()(x)
        assert type(b.mlp.fc1) is Int8Linear
        # four products in a row, about 1 % of noise each
        assert (got - want).norm() <= 0.06 * (want - x).norm()


@pytest.mark.parametrize("watch", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_stochastic_depth_keeps_the_type(dtype, watch):
    """With and without modules called one by one, in training and not."""
    b = block(init_values=None, drop_path=0.4).bfloat16()
    if watch:
        b.norm2.register_forward_hook(lambda *a: None)
    x = torch.randn(3, 512, 128, device=DEV).to(dtype)
    with torch.autocast("cuda", dtype=torch.bfloat16, enabled=dtype == torch.float32):
        assert b.train()(x).dtype == dtype and b.eval()(x).dtype == dtype


@pytest.mark.parametrize("dim, dtype", [(64, torch.float64), (8200, torch.float32), (8192, torch.float32)])
def test_a_block_that_the_norm_kernels_do_not_reach(dim, dtype):
    from test_block_contracts_cpu import Plain
    from speed3r_b200 import forward_blocks

    b = block(dim, mlp_ratio=1 / 64 if dim > 64 else 4.0, attn_class=Plain, init_values=0.3).to(dtype)
    x = torch.randn(2, 5, dim, device=DEV, dtype=dtype)
    with torch.no_grad():
        y, z = b(x), by_modules(b, x)
        # the same PyTorch operations, or at 8192 channels fp32 sums of as many terms in another order
        assert (y - z).norm() <= (0 if dim != 8192 else 8192 * 2.0 ** -24) * z.norm()
        assert torch.equal(forward_blocks([b], x), y)


# ---- 8 bits ----------------------------------------------------------------------------------------------------------------
def test_a_block_in_8_bits_becomes_bf16():
    b = block(init_values=0.1).eval().quantize_int8()
    x = torch.randn(2, 512, 128, device=DEV).bfloat16()
    with torch.no_grad():
        with torch.autocast("cuda", dtype=torch.bfloat16):
            want = b(x.float())
        got = b.bfloat16()(x)
    assert got.dtype == torch.bfloat16 and b.mlp.fc1.weight_scale.dtype == torch.float32
    # parameters of norms and scales in bf16, sums rounded to bf16 three times
    assert (got - want).norm() <= 0.06 * want.norm()


@pytest.mark.parametrize("where", ["attn.qkv", "attn.proj", "attn.gate.0", "mlp.fc1", "mlp.fc2"])
def test_a_block_that_cannot_become_8_bit_stays_as_it_is(where):
    from test_block_contracts_cpu import Adapted

    b = block()
    old = b.get_submodule(where)
    b.set_submodule(where, Adapted(old.in_features, old.out_features).to(DEV))
    kept = {n: type(m) for n, m in b.named_modules()}
    with pytest.raises(RuntimeError, match="something else than a Linear"):
        b.quantize_int8()
    assert {n: type(m) for n, m in b.named_modules()} == kept


# ---- optimiser -------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("fused", [False, True])
def test_a_run_of_pytorchs_adamw_goes_on(fused):
    from speed3r_b200 import AdamW

    make = lambda: [torch.nn.Parameter(torch.linspace(-1, 1, n, device=DEV)) for n in (300, 5000)]
    a, b = make(), make()
    theirs = torch.optim.AdamW(a, lr=1e-2, betas=(0.8, 0.95), fused=fused)
    gen = torch.Generator(device=DEV).manual_seed(0)
    grads = [[torch.randn(p.shape, device=DEV, generator=gen) for p in a] for _ in range(6)]

    def go(params, opt, rounds):
        for gs in rounds:
            for p, g in zip(params, gs):
                p.grad = g.clone()
            opt.step()

    go(a, theirs, grads[:3])
    ours = AdamW(b, lr=1.0)
    ours.load_state_dict(theirs.state_dict())
    for p, q in zip(a, b):
        q.data.copy_(p.data)
    go(a, theirs, grads[3:])
    go(b, ours, grads[3:])
    for p, q in zip(a, b):
        # three steps of lr, each off by a few 2^-23 of itself, and the parameter's own rounding
        assert ((p - q).abs() <= 8 * 2.0 ** -24 * p.abs() + 3 * 1e-2 * 40 * 2.0 ** -24).all()


def test_random_numbers_go_by_seed_and_number():
    def codes(numbers=None, seed=5, count=2):
        p, g, m, v, e, step = state([(2000,)], (True,), seed=3)
        p, g, m, v, e = ([ts[0].clone() for _ in range(count)] for ts in (p, g, m, v, e))       # the same tensor over and over
        ops.adamw_step(p, g, m, v, step, scales=e, seed=seed, numbers=numbers)
        return m

    by_index = codes()
    assert not torch.equal(*by_index) and not torch.equal(*codes([9, 8])) and torch.equal(*codes([7, 7]))
    assert all(torch.equal(a, b) for a, b in zip(by_index, codes([0, 1])))
    assert torch.equal(codes([1, 0])[0], by_index[1]) and torch.equal(codes([1], count=1)[0], by_index[1])
    assert not torch.equal(codes(seed=5 + (1 << 32))[0], by_index[0]) and not torch.equal(codes(seed=5 + (1 << 62))[0], by_index[0])
    for bad in ([0], [0, -1], [0, 1 << 24]):
        with pytest.raises(RuntimeError, match="numbers"):
            codes(bad)


def test_groups_round_by_themselves_and_a_missing_gradient_changes_nothing_else():
    from speed3r_b200 import AdamW

    def run(missing=()):
        ps = [torch.nn.Parameter(torch.linspace(1, 2, 8192, device=DEV).bfloat16()) for _ in range(4)]
        opt = AdamW([dict(params=ps[:2]), dict(params=ps[2:])], lr=1e-3, weight_decay=0.0, state_bits=8)
        for k in range(3):
            for i, p in enumerate(ps):
                p.grad = None if i in missing and k else torch.full_like(p, 0.1)
            opt.step()
        return ps, [opt.state[p]["exp_avg"] for p in ps]

    (ps, ms), (qs, ns) = run(), run(missing=(0, 3))
    assert not torch.equal(ps[0], ps[2]) and not torch.equal(ms[0], ms[2]) and not torch.equal(ms[1], ms[3])
    assert torch.equal(ps[1], qs[1]) and torch.equal(ms[1], ns[1]) and torch.equal(ps[2], qs[2]) and torch.equal(ms[2], ns[2])


@pytest.mark.parametrize("eps", [0.0, 1e-30, 1e-20, 1e-18, 1e-15, 1e-8])
@pytest.mark.parametrize("eight", [False, True])
def test_second_moments_below_the_normal_numbers(eight, eps):
    """Gradients of 1e-19: v is a subnormal number, and its root is what the step is divided by where eps is no larger."""
    from test_gpu_block_ops import values

    n, b1, b2, lr = 5000, 0.9, 0.999, 1e-2
    gen = torch.Generator(device=DEV).manual_seed(4)
    p = torch.randn(n, device=DEV, generator=gen)
    zeros = lambda: torch.zeros(n, device=DEV, dtype=U8 if eight else torch.float32)
    m, v, e, step = zeros(), zeros(), torch.full((2, -(-n // 256)), 27, device=DEV, dtype=U8), torch.zeros((), dtype=torch.int64, device=DEV)
    for t in (1, 2):
        g = (0.5 + 1.5 * torch.rand(n, device=DEV, generator=gen)) * 1e-19
        m0, v0 = (values(m, e[0], 4), values(v, e[1], 5)) if eight else (m.double(), v.double())
        p0, d = p.double(), g.double()
        ops.adamw_step([p], [g], [m], [v], step, lr=lr, betas=(b1, b2), eps=eps, weight_decay=0.0, scales=[e] if eight else None)
        m1, v1 = b1 * m0 + (1 - b1) * d, b2 * v0 + (1 - b2) * d * d
        inv_root = 1 / math.sqrt(1 - b2 ** t)
        root = torch.sqrt(v1) * inv_root + eps
        moved = lr / (1 - b1 ** t) * m1 / root
        # In fp32: b2 v and (1 - b2) g^2 are rounded to multiples of 2^-149, by half a one each, and the square by as little; their sum is
        # exact.  That moves the root by half its share of v, which is within the share itself.  The rest: 2^-24, a few of them.
        share = 2.0 ** -149 * 1.01 / v1
        close = moved.abs() * (40 * 2.0 ** -24 + share) + 8 * 2.0 ** -24 * p0.abs()
        assert p.isfinite().all() and ((p.double() - (p0 - moved)).abs() <= close).all(), (t, eps)


@pytest.mark.parametrize("eight", [False, True])
def test_bf16_parameters_are_rounded_by_all_bits_that_they_drop(eight):
    """Against the same step of fp32 parameters, rounded here."""
    from test_gpu_block_ops import philox

    n, seed = 100_003, 21
    p, g, m, v, e, step = state([(n,)], (eight,), seed=6, dtype=torch.bfloat16)
    wide, m2, v2, e2, step2 = [p[0].float()], [m[0].clone()], [v[0].clone()], [e[0].clone() if eight else None], step.clone()
    ops.adamw_step(wide, g, m2, v2, step2, lr=1e-2, scales=e2)
    ops.adamw_step(p, g, m, v, step, lr=1e-2, scales=e, seed=seed)
    pair = torch.arange((n + 1) // 2, device=DEV)
    low = philox(pair, step.expand(pair.shape), seed)[:n]
    want = ((wide[0].view(torch.int32).long() & 0xFFFFFFFF) + (low >> 16)) >> 16
    assert torch.equal(p[0].view(torch.int16).long() & 0xFFFF, want)


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_updates_far_below_a_bf16_step_happen_on_average(eight, sign):
    """An update of a 8192nd of a step moves one parameter in 8192."""
    n = 1 << 22
    p, g = torch.full((n,), 1.5, device=DEV).bfloat16(), torch.full((n,), sign, device=DEV).bfloat16()
    zeros = lambda: torch.zeros(n, device=DEV, dtype=U8 if eight else torch.float32)
    e = [torch.full((2, n // 256), 27, device=DEV, dtype=U8)] if eight else None
    # the first step is lr in size whatever the gradient
    ops.adamw_step([p], [g], [zeros()], [zeros()], torch.zeros((), dtype=torch.int64, device=DEV), lr=2.0 ** -20, eps=0.0, weight_decay=0.0, scales=e, seed=9)
    step = p.float() - 1.5
    moved = int((step != 0).sum())
    assert ((step == 0) | (step == -sign * 2.0 ** -7)).all()
    # binomial: 512 expected, 22.6 its deviation
    assert abs(moved - n / 8192) <= 6 * math.sqrt(n / 8192)


@pytest.mark.parametrize("bias", [True, False])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("N, K", [(1000, 1024), (257, 500)])
def test_a_token_has_the_same_results_in_every_batch(N, K, dtype, bias):
    """Whichever kernel and tile computes them: bit for bit."""
    gen = torch.Generator(device=DEV).manual_seed(N)
    q, w = (torch.randint(-127, 128, s, device=DEV, dtype=torch.int8, generator=gen) for s in ((9000, K), (N, K)))
    s, ws = (torch.rand(n, device=DEV, generator=gen) + 0.1 for n in (9000, N))
    ws *= 0.01
    b = torch.randn(N, device=DEV, generator=gen) if bias else None
    whole = ops.int8_linear(q, s, w, ws, b, dtype)
    for M in (1, 2, 3, 4, 5, 8, 9, 64, 129, 700):
        assert torch.equal(ops.int8_linear(q[:M], s[:M], w, ws, b, dtype), whole[:M]), M


# ---- norms -----------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("rows", [(3, 50), (40, 1), (2, 5000)])
@pytest.mark.parametrize("wanted", [("d_weight",), ("d_bias", "d_gate_channel"), ("d_scale", "d_post_weight", "d_post_bias"), ("d_gate_channel",),
                                    ("d_weight", "d_bias", "d_scale", "d_post_weight", "d_post_bias", "d_gate_channel")])
def test_sums_that_are_wanted_need_their_own_workspace_and_no_more(rows, wanted):
    """Through the library's C entry, with just the workspace that the header asks for: the same sums, nothing behind it written."""
    import ctypes as C
    from speed3r_b200 import _lib
    from test_block_contracts_cpu import SUMS, norm_backward_args

    B, T, Ch = *rows, 64
    gen = torch.Generator(device=DEV).manual_seed(B)
    rand = lambda *s: torch.randn(*s, device=DEV, generator=gen)
    t = {n: rand(B * T, Ch) for n in ("r", "y", "dr", "dh", "dx")}
    t |= {n: rand(Ch) for n in ("weight", "bias", "scale", "post_weight", "post_bias")} | dict(gate=rand(B, Ch), stats=rand(4, B * T))
    lib = _lib.load()
    whole = lib.s3r_residual_norm_bwd_workspace_bytes(B, T, Ch, 2)

    def sums(names):
        need = whole // 6 * len(names)
        space = torch.full((need + 4096,), 7, dtype=U8, device=DEV)
        out = {n: torch.zeros(B, Ch, device=DEV) if n == "d_gate_channel" else torch.zeros(Ch, device=DEV) for n in names}
        f, g = norm_backward_args(0, (), batch=B, tokens=T, **{n: t[n].data_ptr() for n in ("r", "y", "weight", "bias", "scale", "post_weight", "post_bias", "gate", "stats")},
                                  x=t["r"].data_ptr())
        g.dr, g.dh, g.dx, g.workspace, g.workspace_bytes = (*(t[n].data_ptr() for n in ("dr", "dh", "dx")), space.data_ptr(), need)
        for n, o in out.items():
            setattr(g, n, o.data_ptr())
        assert lib.s3r_residual_norm_bwd(C.byref(f), C.byref(g), torch.cuda.current_stream().cuda_stream) == 0
        torch.cuda.synchronize()
        assert (space[need:] == 7).all()
        return out

    every = sums(SUMS)
    assert all(o.isfinite().all() and (o != 0).any() for o in every.values())
    got = sums(wanted)
    assert all(torch.equal(got[n], every[n]) for n in wanted)


@pytest.mark.parametrize("learn", [(), ("gate",)])
def test_backward_takes_no_memory_for_sums_that_nobody_wants(learn):
    B, Ch = 8192, 1024
    x, y = (torch.randn(B, 1, Ch, device=DEV).requires_grad_(True) for _ in range(2))
    gate = torch.randn(B, 1, Ch, device=DEV).requires_grad_("gate" in learn)
    r, h = ops.residual_norm(x, y, (torch.ones(Ch, device=DEV), None, 1e-5), gate=gate)
    leaves = [x, y] + [gate] * len(learn)
    grads = [torch.ones_like(t) for t in (r, h)]
    one = B * Ch * 4
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    torch.autograd.grad((r, h), leaves, grads)
    torch.cuda.synchronize()
    # dx and dy; with the gate its gradient, and a sum per entry of it
    assert torch.cuda.max_memory_allocated() - before <= (2 + 2 * len(learn)) * one + (8 << 20)


def saved_by(call):
    """Addresses of the tensors that autograd keeps of a call."""
    kept = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: kept.append(t.data_ptr()) or t, lambda t: t):
        out = call()
    return set(kept), out


@pytest.mark.parametrize("learn", ["", "scale", "gate", "post"])
def test_the_branch_is_kept_where_it_is_needed_and_only_there(learn):
    x, y = (torch.randn(2, 33, 256, device=DEV).to(t).requires_grad_(True) for t in (torch.float32, torch.bfloat16))
    w, scale, gate = (torch.randn(s, device=DEV).requires_grad_(n == learn) for n, s in (("w", 256), ("scale", 256), ("gate", (2, 33, 1))))
    kept, (r, h) = saved_by(lambda: ops.residual_norm(x, y, (w, None, 1e-5), scale, gate, (None, None, 1e-5) if learn == "post" else None))
    assert (y.data_ptr() in kept) == bool(learn)
    assert r.data_ptr() in kept and x.data_ptr() not in kept and h.data_ptr() not in kept


@pytest.mark.parametrize("C, rows", [(64, 9500), (100, 9473), (132, 9999), (256, 9472), (320, 5000), (1024, 2371), (2056, 601), (3000, 592), (4096, 777)])
@pytest.mark.parametrize("kw", [dict(kind="rms"), dict(gate="channel"), dict(gate="channel", kind="rms", post=True), dict(branch=False), dict(branch=False, kind="rms"),
                                dict(half=True), dict(half=True, gate="token", post=True), dict(norm=False)], ids=str)
def test_norms_of_many_rows(C, rows, kw):
    """As many as the kernel whose CTAs stay is for (four rows and more for each group that is resident), in every form."""
    from test_gpu_block_ops import Norm

    kw = dict(kw)
    gate = {None: None, "channel": (2, 1, C), "token": (2, -(-rows // 2), 1)}[kw.pop("gate", None)]
    types = dict.fromkeys("xyhw", torch.float16) if kw.pop("half", False) else {}
    n = Norm((2, -(-rows // 2), C), gate=gate, seed=C, **types, **kw)
    n.train()
    if not kw.get("norm", True):
        return
    n.h_type = torch.float32
    with torch.no_grad():
        r, h = n.call()
        r8, q, s = ops.residual_norm_int8(n.x, n.y, n.norm, n.scale, n.gate, n.post, n.kind)
        q2, s2 = ops.quantize_tokens(h)
    assert torch.equal(r8, r) and torch.equal(q, q2) and torch.equal(s, s2)


def test_a_step_that_makes_states_is_not_captured():
    """Its replays would begin anew each time."""
    from speed3r_b200 import AdamW

    def captured(opt):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            opt.step()
        return graph

    ps = [torch.nn.Parameter(torch.ones(300, device=DEV)) for _ in range(2)]
    for p in ps:
        p.grad = torch.ones_like(p)
    opt = AdamW(ps, lr=0.1)
    with pytest.raises(RuntimeError, match="first step cannot be captured"):
        captured(opt)
    opt = AdamW(ps, lr=0.1)
    opt.step()
    grad, ps[1].grad = ps[1].grad, None
    with pytest.raises(RuntimeError, match="left out for the first time"):
        captured(opt)
    opt.step()                                          # outside of the graph it is taken
    captured(opt).replay()
    assert [int(opt.state[p]["step"]) for p in ps] == [3, 1]
    ps[1].grad = grad
    captured(opt).replay()
    assert [int(opt.state[p]["step"]) for p in ps] == [4, 2]


@pytest.mark.parametrize("what", ["params", "exp_avg", "exp_avg_sq", "scales", "scales of m and v"])
def test_memory_that_is_listed_twice_in_part_is_refused(what):
    p, g, m, v, e, step = state([(512,), (512,)], (True, True))
    flat = torch.zeros(4096, device=DEV)
    if what == "params":
        p = [flat[:512], flat[511:1023]]
    elif what == "scales":
        e = [e[0], e[0]]
    elif what == "scales of m and v":
        whole = torch.zeros(2, 4, device=DEV, dtype=U8)
        e = [whole[:, :2], whole[:, 1:3]]
    else:
        codes = flat.view(U8)
        (m if what == "exp_avg" else v)[:] = [codes[:512], codes[100:612]]
    with pytest.raises(RuntimeError, match="listed twice"):
        ops.adamw_step(p, g, m, v, step, scales=e)
    assert int(step) == 3
    if what == "params":                                 # side by side they may lie
        ops.adamw_step([flat[:512], flat[512:1024]], g, m, v, step, scales=e)
