"""What the operators around the attention promise to tracers, to autograd and to whoever calls them, as far as no GPU is needed."""
import pytest
import torch

from speed3r_b200 import ops

U8 = torch.uint8


def raises(text, call):
    with pytest.raises(RuntimeError, match=text):
        call()


# ---- tracing ---------------------------------------------------------------------------------------------------------------
def traced(f, *args):
    """The graph that ahead-of-time autograd makes of f(*args).  Tracing reads shapes only; what is traced is not run."""
    from torch._functorch.aot_autograd import aot_module_simplified

    class Seen(Exception):
        pass

    graphs = []

    def keep(graph, inputs):
        graphs.append(graph.graph)
        raise Seen

    ops._ops()
    torch._dynamo.reset()
    with pytest.raises(Exception):                       # Seen, as the compiler passes it on
        torch.compile(f, backend=lambda gm, ins: aot_module_simplified(gm, ins, fw_compiler=keep), fullgraph=True)(*args)
    return graphs[0]


def behind(node, earlier):
    """Whether `node` depends on `earlier`."""
    seen, todo = set(), [node]
    while todo:
        n = todo.pop()
        if n is earlier:
            return True
        if n not in seen:
            seen.add(n)
            todo += n.all_input_nodes
    return False


def test_step_is_traced_as_writing_everything_that_it_writes():
    n = 300
    m, v = (torch.zeros(n, dtype=U8) for _ in range(2))
    scales, step = torch.zeros(2, 2, dtype=U8), torch.zeros((), dtype=torch.int64)
    names = ("p", "m", "v", "scales", "step", "p of 32-bit states", "m of 32 bits", "v of 32 bits")

    def f(g, p, m, v, scales, step, q, m32, v32):
        written = (p, m, v, scales, step, q, m32, v32)
        before = [t + 1 for t in written]
        ops.adamw_step([p, q], [g, g], [m, m32], [v, v32], step, scales=[scales, None])
        return [t * 2 for t in before] + [t + 1 for t in written]

    graph = traced(f, torch.ones(n), torch.zeros(n), m, v, scales, step, *(torch.zeros(n) for _ in range(3)))
    the_step = [node for node in graph.nodes if node.op == "call_function" and "auto_functionalized" in str(node.target)]
    assert len(the_step) == 1
    out = next(node for node in graph.nodes if node.op == "output").args[0][-2 * len(names):]
    for name, before, after in zip(names, out, out[len(names):]):
        assert not behind(before, the_step[0]), name
        assert behind(after, the_step[0]), name


# ---- forward mode ----------------------------------------------------------------------------------------------------------
def test_tangents_are_refused_and_not_dropped():
    """In every operator and every floating argument, before anything is computed."""
    import torch.autograd.forward_ad as fwd

    x, q, s = torch.zeros(4, 8), torch.zeros(4, 8, dtype=torch.int8), torch.ones(4)
    codes, scales = torch.zeros(32, dtype=U8), torch.zeros(2, 1, dtype=U8)
    step = torch.zeros((), dtype=torch.int64)
    with fwd.dual_level():
        dual = lambda t: fwd.make_dual(t.clone(), torch.ones_like(t))
        d, one = dual(x), dual(torch.ones(()))
        calls = [lambda: ops.residual_norm(d, None, (None, None, 1e-5)), lambda: ops.residual_norm(x, d), lambda: ops.residual_norm(x, x, scale=dual(torch.ones(8))),
                 lambda: ops.residual_norm_int8(d, None, (None, None, 1e-5)), lambda: ops.quantize_tokens(d),
                 lambda: ops.int8_linear(q, dual(s), q, s), lambda: ops.int8_linear(q, s, q, dual(s)), lambda: ops.int8_linear(q, s, q, s, dual(s)),
                 lambda: ops.grad_norm([x, d]),
                 lambda: ops.adamw_step([x], [x], [x], [x], step, lr=one), lambda: ops.adamw_step([x], [x], [x], [x], step, grad_norm=one)]
        calls += [lambda i=i: ops.adamw_step(*[[x, d if k == i else x] for k in range(4)], step) for i in range(4)]
        calls += [lambda i=i: ops.adamw_state([codes], [codes], [scales], out=[[dual(torch.zeros(32)) if k == i else torch.zeros(32)] for k in range(2)]) for i in range(2)]
        for i, call in enumerate(calls):
            with pytest.raises(NotImplementedError, match="forward mode"):
                call()
                pytest.fail(f"call {i} went through")


# ---- the block -------------------------------------------------------------------------------------------------------------
def test_a_scale_of_another_formula_is_called():
    """What has a parameter named gamma need not multiply with it."""
    from speed3r_b200 import BlockRope
    from speed3r_b200.block import LayerScale

    class Exponential(LayerScale):
        def forward(self, x):
            return x * self.gamma.exp()

    class Named(torch.nn.Identity):
        gamma = torch.full((64,), 3.0)

    class Own(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.gamma = torch.nn.Parameter(torch.ones(64))

        def forward(self, x):
            return x + self.gamma

    b = BlockRope(64, 1, init_values=0.1)
    assert b._fuses()
    for name in ("ls1", "ls2"):
        for other in (Exponential(64), Named(), Own()):
            b = BlockRope(64, 1, init_values=0.1)
            setattr(b, name, other)
            assert not b._fuses(), other
    b = BlockRope(64, 1)
    b.ls1.gamma = torch.full((64,), 3.0)                # an Identity stays one
    assert b._fuses() and b._scale(b.ls1) is None


class Gated(torch.nn.Module):
    """A feed-forward layer of three matrices."""

    def __init__(self, in_features, hidden_features=None, out_features=None, act_layer=None, drop=0.0, bias=True):
        super().__init__()
        hidden_features = hidden_features or in_features
        self.w12 = torch.nn.Linear(in_features, 2 * hidden_features, bias=bias)
        self.w3 = torch.nn.Linear(hidden_features, out_features or in_features, bias=bias)

    def forward(self, x):
        a, b = self.w12(x).chunk(2, -1)
        return self.w3(torch.nn.functional.silu(a) * b)


def test_a_feed_forward_layer_of_other_matrices_in_8_bits_raises_and_nothing_changes():
    from speed3r_b200 import BlockRope
    b = BlockRope(64, 1, ffn_layer=Gated)
    kept = {n: type(m) for n, m in b.named_modules()}
    raises("not an MLP of two Linears", b.quantize_int8)
    assert {n: type(m) for n, m in b.named_modules()} == kept
    assert not b._mlp_takes_int8()


class Plain(torch.nn.Module):
    """An attention that runs anywhere."""

    def __init__(self, dim, num_heads, **kw):
        super().__init__()
        self.lin = torch.nn.Linear(dim, dim)

    def forward(self, x, xpos=None):
        return self.lin(x)


@pytest.mark.parametrize("dim, dtype", [(64, torch.float32), (64, torch.float64), (8200, torch.float32), (64, torch.bfloat16)])
def test_a_block_that_the_kernels_do_not_reach_is_computed_by_its_modules(dim, dtype):
    from speed3r_b200 import BlockRope, forward_blocks
    torch.manual_seed(0)
    b = BlockRope(dim, 1, mlp_ratio=1 / 64 if dim > 64 else 4.0, attn_class=Plain, init_values=0.3).to(dtype)
    x = torch.randn(2, 5, dim, dtype=dtype)
    y = x + b.ls1(b.attn(b.norm1(x)))
    y = y + b.ls2(b.mlp(b.norm2(y)))
    assert torch.equal(b(x), y) and torch.equal(forward_blocks([b], x), y) and y.dtype == dtype


def test_stochastic_depth_keeps_the_type_of_the_branch():
    from speed3r_b200 import BlockRope
    b = BlockRope(64, 1, attn_class=Plain, drop_path=0.4).bfloat16().train()
    assert b(torch.randn(3, 5, 64).bfloat16()).dtype == torch.bfloat16


# ---- 8 bits ----------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("change", [lambda m: m.bfloat16(), lambda m: m.half(), lambda m: m.double(), lambda m: m.to(torch.bfloat16), lambda m: m.to("cpu", torch.float16)])
def test_scales_of_an_8_bit_linear_stay_fp32(change):
    from speed3r_b200 import Int8Linear
    scale, bias = torch.rand(5) + 0.1, torch.randn(5)
    m = torch.nn.Sequential(Int8Linear(torch.zeros(5, 16, dtype=torch.int8), scale.clone(), bias.clone()), torch.nn.Linear(5, 5))
    change(m)
    assert torch.equal(m[0].weight_scale, scale) and torch.equal(m[0].bias, bias) and m[0].weight.dtype == torch.int8
    assert m[0].weight_scale.dtype == m[0].bias.dtype == torch.float32 and m[1].weight.dtype != torch.float32
    assert set(m.state_dict()) == {"0.weight", "0.weight_scale", "0.bias", "1.weight", "1.bias"}
    assert Int8Linear(torch.zeros(5, 16, dtype=torch.int8), scale, None).half().bias is None
    assert m.to("meta")[0].weight_scale.device.type == "meta"


class Adapted(torch.nn.Linear):
    """A Linear with something beside it, as fine-tuning adds."""

    def forward(self, x):
        return super().forward(x) + x.sum(-1, keepdim=True)


def test_what_is_more_than_a_linear_does_not_become_an_8_bit_one():
    from speed3r_b200 import BlockRope, Int8Linear
    raises("something else than a Linear", lambda: Int8Linear.of(Adapted(16, 5)))
    raises("something else than a Linear", lambda: Int8Linear.of(torch.nn.Identity()))
    wrapped = torch.nn.Linear(16, 5)
    wrapped.forward = lambda x: x
    raises("something else than a Linear", lambda: Int8Linear.of(wrapped))


# ---- optimiser -------------------------------------------------------------------------------------------------------------
def stepped(params, steps=3, **kw):
    """torch.optim.AdamW after some steps, some parameters from the second on."""
    opt = torch.optim.AdamW(params, **kw)
    for i in range(steps):
        for k, p in enumerate(params):
            p.grad = torch.full_like(p, 0.1 * (k + 1)) if i or k else None
        opt.step()
    return opt


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_state_dict_of_pytorchs_adamw_loads(dtype):
    from speed3r_b200 import AdamW
    make = lambda: [torch.nn.Parameter(torch.ones(3, 4, dtype=dtype)), torch.nn.Parameter(torch.ones(5, dtype=dtype))]
    theirs = stepped(make(), lr=2e-3, betas=(0.8, 0.9), weight_decay=0.3)
    saved = theirs.state_dict()
    params = make()
    opt = AdamW(params, lr=1.0, state_bits=8, seed=7)
    opt.load_state_dict(saved)
    (group,) = opt.param_groups
    assert (group["lr"], group["betas"], group["weight_decay"]) == (2e-3, (0.8, 0.9), 0.3)
    assert (group["state_bits"], group["min_8bit_size"], group["seed"]) == (8, 4096, 7)
    for p, i in zip(params, range(2)):
        st, want = opt.state[p], saved["state"][i]
        assert st["step"].dtype == torch.int64 and int(st["step"]) == int(want["step"]) == 2 + i
        for name in ("exp_avg", "exp_avg_sq"):
            assert st[name].dtype == torch.float32 and torch.equal(st[name], want[name].float()) and st[name].data_ptr() != want[name].data_ptr()
    # as older versions save it: the count as a number
    old = {"state": {i: {**st, "step": int(st["step"])} for i, st in saved["state"].items()}, "param_groups": saved["param_groups"]}
    opt.load_state_dict(old)
    assert [int(opt.state[p]["step"]) for p in params] == [2, 3] and opt.state[params[0]]["step"].dtype == torch.int64


@pytest.mark.parametrize("name", ["maximize", "amsgrad"])
def test_a_state_dict_of_another_formula_is_refused(name):
    from speed3r_b200 import AdamW
    make = lambda: [torch.nn.Parameter(torch.ones(3))]
    saved = stepped(make(), **{name: True}).state_dict()
    params = make()
    opt = AdamW(params, lr=0.5)
    raises(name, lambda: opt.load_state_dict(saved))
    assert opt.param_groups[0]["lr"] == 0.5 and not opt.state


def test_numbers_of_a_step_are_checked_without_a_gpu(lib):
    import ctypes as C
    from test_block_ops_cpu import AdamArgs

    buf = C.create_string_buffer(4096)
    p = (C.addressof(buf) + 255) & ~255
    one, count, types = (C.c_void_p * 1)(p), (C.c_int64 * 1)(4), (C.c_int * 1)(0)
    at = lambda x: C.cast(x, C.c_void_p)
    a = AdamArgs(n=1, params=at(one), grads=at(one), m=at(one), v=at(one), counts=at(count), param_types=at(types), grad_types=at(types), step=p,
                 lr_host=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, seed=1, workspace=p)
    assert lib.s3r_adamw_step_numbered(None, None, None) == -4
    assert lib.s3r_adamw_step_numbered(C.byref(a), at((C.c_uint32 * 1)(1 << 24)), None) == -6


def test_the_optimiser_numbers_its_parameters(monkeypatch):
    """Over all groups, whichever of them have a gradient and however many calls a step makes."""
    from speed3r_b200 import AdamW
    seen = []
    monkeypatch.setattr(ops, "adamw_step", lambda params, *a, numbers=None, **kw: seen.extend(zip([id(p) for p in params], numbers or [None] * len(params))))
    ps = [torch.nn.Parameter(torch.ones(3)) for _ in range(5)]
    opt = AdamW([dict(params=ps[:3]), dict(params=ps[3:], weight_decay=0.0)])
    for missing in ((), (0,), (1, 3), ()):
        for i, p in enumerate(ps):
            p.grad = None if i in missing else torch.ones(3)
        seen.clear()
        opt.step()
        assert sorted(seen) == sorted((id(p), i) for i, p in enumerate(ps) if i not in missing)
    opt = AdamW(ps, seed=None)
    seen.clear()
    opt.step()
    assert [n for _, n in seen] == [None] * 5


def test_an_eps_that_fp32_does_not_hold_is_refused(lib):
    import ctypes as C
    from test_block_ops_cpu import AdamArgs

    buf = C.create_string_buffer(4096)
    p = (C.addressof(buf) + 255) & ~255
    a = AdamArgs(n=-1, step=p, lr_host=1e-3, beta1=0.9, beta2=0.999, workspace=p)
    for eps, code in ((0.0, -1), (2.0 ** -126, -1), (1e-8, -1), (1e-38, -2), (1e-60, -2), (-1.0, -2), (float("nan"), -2)):
        a.eps, a.n = eps, 0 if code == -2 else -1
        assert lib.s3r_adamw_step(C.byref(a), None) == code, eps


def test_rows_whose_columns_an_int_does_not_reach_are_refused(lib):
    """The last column's successor in a thread's walk has to be a column number too."""
    p = 1 << 12
    rc = lambda channels: lib.s3r_quantize_rows(p, 0, 1 << 31, p, 1 << 31, p, 1, channels, None)
    assert rc(2 ** 31 - 1) == -6 and rc(2 ** 31 - 8192) == -6


def norm_backward_args(p, wanted, **kw):
    """Arguments of a backward whose tensors all lie at `p`, with the named sums wanted."""
    import ctypes as C
    from test_block_ops_cpu import NormArgs

    class Grad(C.Structure):
        _fields_ = [(n, C.c_void_p) for n in ("dr", "dh", "dx", "dy", "d_weight", "d_bias", "d_scale", "d_post_weight", "d_post_bias", "d_gate_row", "d_gate_channel",
                                              "workspace")] + [("workspace_bytes", C.c_size_t)]

    f = NormArgs(batch=3, tokens=50, channels=64, post=1, x=p, y=p, r=p, stats=p, weight=p, bias=p, scale=p, post_weight=p, post_bias=p, gate=p, gate_mode=2,
                 gate_stride_b=64)
    for k, v in kw.items():
        setattr(f, k, v)
    return f, Grad(dr=p, dh=p, dx=p, workspace=p, **{n: p for n in wanted})


SUMS = ("d_weight", "d_bias", "d_scale", "d_post_weight", "d_post_bias", "d_gate_channel")


@pytest.mark.parametrize("count", range(1, 7))
def test_a_workspace_that_is_too_small_for_the_sums_is_refused(lib, count):
    import ctypes as C
    f, g = norm_backward_args(1 << 12, SUMS[:count])
    whole = lib.s3r_residual_norm_bwd_workspace_bytes(3, 50, 64, 2)
    assert whole > 0 and whole % 6 == 0
    g.workspace_bytes = whole // 6 * count - 1
    assert lib.s3r_residual_norm_bwd(C.byref(f), C.byref(g), None) == -6


def test_copies_of_the_optimiser_clip_too(monkeypatch):
    import copy
    import pickle
    from speed3r_b200 import AdamW

    seen = []
    monkeypatch.setattr(ops, "grad_norm", lambda grads: torch.tensor(3.0))
    monkeypatch.setattr(ops, "adamw_step", lambda *a, grad_norm=None, max_norm=None, **kw: seen.append((float(grad_norm), max_norm)))
    p = torch.nn.Parameter(torch.ones(3))
    opt = AdamW([p], max_norm=2.0)
    for other in (copy.deepcopy(opt), pickle.loads(pickle.dumps(opt))):
        (q,) = other.param_groups[0]["params"]
        q.grad = torch.ones(3)
        other.step()
    assert seen == [(3.0, 2.0)] * 2


def test_another_attention_is_given_activations_in_8_bits_too():
    from speed3r_b200 import BlockRope, Int8Linear, SparseFlashAttentionRope

    class Other(SparseFlashAttentionRope):
        def forward(self, x, attn_bias=None, xpos=None):
            return super().forward(x * 1.0, attn_bias, xpos)

    for cls in (Other, Plain, SparseFlashAttentionRope):
        b = BlockRope(64, 1, attn_class=cls)
        assert not b._takes_int8()
        b.attn.qkv = Int8Linear(torch.zeros(192, 64, dtype=torch.int8), torch.ones(192), None)
        assert b._takes_int8() == (cls is SparseFlashAttentionRope)


@pytest.mark.filterwarnings("ignore::FutureWarning")
def test_a_linear_with_hooks_does_not_become_an_8_bit_one():
    """One whose weight a hook makes of others has, until it is called, the weight of before."""
    from speed3r_b200 import Int8Linear
    normed = torch.nn.utils.weight_norm(torch.nn.Linear(16, 5))
    with torch.no_grad():
        normed.weight_g.mul_(3)
    raises("has hooks", lambda: Int8Linear.of(normed))
    watched = torch.nn.Linear(16, 5)
    handle = watched.register_forward_hook(lambda m, i, o: o * 2)
    raises("has hooks", lambda: Int8Linear.of(torch.nn.Linear(16, 5), watched))
    handle.remove()
    raises("no CPU path", lambda: Int8Linear.of(watched))
