"""What the operators of the dense half of a block refuse, and what they promise to tracers, as far as no GPU is needed."""
import ctypes as C

import pytest
import torch

from speed3r_b200 import ops

BF16 = torch.bfloat16


def raises(text, call, error=RuntimeError):
    with pytest.raises(error, match=text):
        call()


# ---- calls that are refused ------------------------------------------------------------------------------------------------
def test_cpu_tensors_are_refused():
    x, w = torch.zeros(4, 8, dtype=BF16), torch.zeros(16, 8, dtype=BF16)
    raises("CUDA", lambda: ops.linear(x, w))
    raises("CUDA", lambda: ops.linear(x.requires_grad_(True), w, act="gelu"))
    raises("CUDA", lambda: ops.qkv_norm_rope(torch.zeros(1, 4, 3 * 64, dtype=BF16), 1))


def test_names_are_checked():
    x, w = torch.zeros(4, 8, dtype=BF16), torch.zeros(16, 8, dtype=BF16)
    raises("act must be", lambda: ops.linear(x, w, act="relu"))
    raises("out_dtype must be", lambda: ops.linear(x, w, out_dtype=torch.float64))
    raises("kind must be", lambda: ops.qkv_norm_rope(torch.zeros(1, 4, 192), 1, kind="batch"))


def test_rotations_are_checked():
    """In front of everything that needs a GPU."""
    x = torch.zeros(2, 4, 3 * 64)
    pos, table = torch.zeros(2, 4, 2, dtype=torch.int64), torch.zeros(8, 16)
    raises("come together", lambda: ops.qkv_norm_rope(x, 1, pos=pos))
    raises("come together", lambda: ops.qkv_norm_rope(x, 1, cos=table, sin=table))
    raises("int64 or int32", lambda: ops.qkv_norm_rope(x, 1, pos=pos.float(), cos=table, sin=table))
    raises("pos must be", lambda: ops.qkv_norm_rope(x, 1, pos=pos[:, :3], cos=table, sin=table))
    raises("pos must be", lambda: ops.qkv_norm_rope(x, 1, pos=torch.zeros(3, 4, 2, dtype=torch.int64), cos=table, sin=table))
    raises("no gradients", lambda: ops.qkv_norm_rope(x, 1, pos=pos, cos=table.clone().requires_grad_(True), sin=table))
    raises("batch, tokens, channels", lambda: ops.qkv_norm_rope(x[0], 1))


def test_forward_mode_is_refused():
    import torch.autograd.forward_ad as fwd

    x, w, s = torch.zeros(4, 8, dtype=BF16), torch.zeros(8, 8, dtype=BF16), torch.ones(8)
    qkv, n = torch.zeros(1, 4, 24), torch.ones(8)
    pos, table = torch.zeros(1, 4, 1, dtype=torch.int64), torch.zeros(8, 4)
    with fwd.dual_level():
        dual = lambda t: fwd.make_dual(t.clone(), torch.ones_like(t))
        calls = [lambda: ops.linear(dual(x), w), lambda: ops.linear(x, dual(w)), lambda: ops.linear(x, w, dual(s)), lambda: ops.linear(x, w, scale=dual(s)),
                 lambda: ops.linear(x, w, residual=dual(x)), lambda: ops.qkv_norm_rope(dual(qkv), 1), lambda: ops.qkv_norm_rope(qkv, 1, q_norm=(dual(n), None, 1e-5)),
                 lambda: ops.qkv_norm_rope(qkv, 1, k_norm=(n, dual(n), 1e-5)), lambda: ops.qkv_norm_rope(qkv, 1, pos=pos, cos=dual(table), sin=table)]
        for call in calls:
            raises("forward mode", call, NotImplementedError)


# ---- shapes on meta tensors, tracing ---------------------------------------------------------------------------------------
def meta(*shape, dtype=BF16):
    return torch.zeros(*shape, dtype=dtype, device="meta")


def test_shapes():
    x, w = meta(2, 5, 40), meta(24, 40)
    assert ops.linear(x, w).shape == (2, 5, 24) and ops.linear(x, w).dtype == BF16
    assert ops.linear(x, w, residual=meta(2, 5, 24, dtype=torch.float32)).dtype == torch.float32
    leaves = [x.requires_grad_(True), w.requires_grad_(True), meta(24, dtype=torch.float32).requires_grad_(True), meta(24).requires_grad_(True),
              meta(2, 5, 24, dtype=torch.float32).requires_grad_(True)]
    y = ops.linear(leaves[0], leaves[1], leaves[2], "gelu", leaves[4], leaves[3])
    for g, t in zip(torch.autograd.grad(y, leaves, torch.zeros_like(y)), leaves):
        assert g.shape == t.shape and g.dtype == t.dtype
    qkv, n = meta(2, 7, (4 + 2 * 2) * 48).requires_grad_(True), [meta(48, dtype=torch.float32).requires_grad_(True) for _ in range(4)]
    out = ops.qkv_norm_rope(qkv, 4, 2, q_norm=(n[0], n[1], 1e-5), k_norm=(n[2], n[3], 1e-5))
    assert [tuple(o.shape) for o in out] == [(2, 4, 7, 48), (2, 2, 7, 48), (2, 2, 7, 48)]
    for g, t in zip(torch.autograd.grad(out, [qkv] + n, [torch.zeros_like(o) for o in out]), [qkv] + n):
        assert g.shape == t.shape and g.dtype == t.dtype


def test_second_derivatives_are_refused():
    x, w = meta(5, 40).requires_grad_(True), meta(24, 40)
    y = ops.linear(x, w, act="silu")
    (g,) = torch.autograd.grad(y, x, torch.zeros_like(y), create_graph=True)
    raises("cannot be differentiated again", lambda: torch.autograd.grad(g, x, torch.zeros_like(g)))
    x = meta(1, 5, 192).requires_grad_(True)
    q, k, v = ops.qkv_norm_rope(x, 1, q_norm=(None, None, 1e-5))
    (g,) = torch.autograd.grad(q, x, torch.zeros_like(q), create_graph=True)
    raises("cannot be differentiated again", lambda: torch.autograd.grad(g, x, torch.zeros_like(g)))


def test_operators_are_traced():
    """As one node each, forward and backward."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx

    def f(x, w, b, qkv, n):
        y = ops.linear(x, w, b, "gelu")
        q, k, v = ops.qkv_norm_rope(qkv, 2, 1, q_norm=(n, None, 1e-5))
        return torch.autograd.grad([y, q], [x, w, b, qkv, n], [torch.ones_like(y), torch.ones_like(q)])

    with FakeTensorMode():
        make = lambda *s, t=BF16: torch.zeros(*s, dtype=t).requires_grad_(True)
        graph = make_fx(f)(make(4, 8), make(16, 8), make(16, t=torch.float32), make(1, 4, 4 * 8), make(8, t=torch.float32))
    names = [str(n.target) for n in graph.graph.nodes if n.op == "call_function"]
    for want in ("linear_fwd", "linear_bwd", "qkv_norm_rope_fwd", "qkv_norm_rope_bwd"):
        assert sum(f"speed3r_b200.{want}." in n for n in names) == 1, (want, names)


# ---- the C ABI ------------------------------------------------------------------------------------------------------------------
class LinearArgs(C.Structure):
    _fields_ = [("M", C.c_int64), ("N", C.c_int), ("K", C.c_int), ("type", C.c_int), ("x", C.c_void_p), ("x_pitch", C.c_int64), ("weight", C.c_void_p),
                ("w_pitch", C.c_int64), ("bias", C.c_void_p), ("scale", C.c_void_p), ("residual", C.c_void_p), ("bias_type", C.c_int), ("scale_type", C.c_int),
                ("residual_type", C.c_int), ("act", C.c_int), ("out", C.c_void_p), ("out_type", C.c_int), ("workspace", C.c_void_p), ("workspace_bytes", C.c_size_t)]


class LinearGrad(C.Structure):
    _fields_ = [("dy", C.c_void_p), ("dz", C.c_void_p), ("dz_pitch", C.c_int64), ("d_bias", C.c_void_p), ("d_scale", C.c_void_p), ("workspace", C.c_void_p),
                ("workspace_bytes", C.c_size_t)]


class RopeArgs(C.Structure):
    _fields_ = ([("batch", C.c_int64), ("tokens", C.c_int64)] + [(n, C.c_int) for n in ("heads", "kv_heads", "head_dim", "kind", "q_normed", "k_normed")] +
                [("q_eps", C.c_float), ("k_eps", C.c_float)] + [(n, C.c_int) for n in ("type", "param_type", "table_type", "axes", "pairs", "rows")] +
                [(n, C.c_int64) for n in ("stride_b", "stride_t", "pos_stride_b", "pos_stride_t", "cos_pitch", "sin_pitch")] +
                [(n, C.c_void_p) for n in ("qkv", "pos", "cos", "sin", "q_weight", "q_bias", "k_weight", "k_bias", "q", "k", "v")])


class RopeGrad(C.Structure):
    _fields_ = ([(n, C.c_void_p) for n in ("dq", "dk", "dv")] + [(n, C.c_int64 * 3) for n in ("dq_strides", "dk_strides", "dv_strides")] +
                [(n, C.c_void_p) for n in ("d_qkv", "d_q_weight", "d_q_bias", "d_k_weight", "d_k_bias", "workspace")] + [("workspace_bytes", C.c_size_t)])


NULL, UNSUPPORTED, ALIGNMENT, SHAPE, TOO_LARGE = -4, -2, -3, -1, -6
P = 0x7F0000000000        # never read: every call below is refused


def linear_args(**more):
    return LinearArgs(**{**dict(M=64, N=32, K=40, type=1, x=P, x_pitch=40, weight=P, w_pitch=40, out=P, out_type=1), **more})


@pytest.mark.parametrize("more, code", [
    (dict(x=None), NULL), (dict(weight=None), NULL), (dict(out=None), NULL), (dict(M=0), SHAPE), (dict(N=0), SHAPE), (dict(K=-1), SHAPE), (dict(x_pitch=32), SHAPE),
    (dict(w_pitch=39), SHAPE), (dict(type=0), UNSUPPORTED), (dict(type=3), UNSUPPORTED), (dict(out_type=5), UNSUPPORTED), (dict(act=4), UNSUPPORTED), (dict(act=-1), UNSUPPORTED),
    (dict(bias=P, bias_type=7), UNSUPPORTED), (dict(scale=P, scale_type=-1), UNSUPPORTED), (dict(residual=P, residual_type=3), UNSUPPORTED), (dict(x=P + 8), ALIGNMENT),
    (dict(x_pitch=44), ALIGNMENT), (dict(weight=P + 2), ALIGNMENT), (dict(bias=P + 2), ALIGNMENT), (dict(residual=P + 1, residual_type=1), ALIGNMENT), (dict(out=P + 1), ALIGNMENT),
    (dict(M=1 << 31), TOO_LARGE)])
def test_c_abi_refuses_linear(lib, more, code):
    assert lib.s3r_linear_fwd(C.byref(linear_args(**more)), None) == code


def test_c_abi_refuses_linear_gradients(lib):
    f = linear_args(bias=P)
    back = lambda f=f, **g: lib.s3r_linear_bwd(C.byref(f), C.byref(LinearGrad(**{**dict(dy=P, dz=P, dz_pitch=32), **g})), None)
    need = lib.s3r_linear_bwd_workspace_bytes(64, 32)
    assert need == 2 * 32 * 4 and lib.s3r_linear_bwd_workspace_bytes(0, 32) == 0
    assert lib.s3r_linear_bwd(C.byref(f), None, None) == NULL and lib.s3r_linear_bwd(None, None, None) == NULL
    assert back(dy=None) == NULL and back(dz_pitch=24) == ALIGNMENT and back(dz=P + 8) == ALIGNMENT and back(dy=P + 1) == ALIGNMENT
    assert back(d_bias=P) == TOO_LARGE and back(d_bias=P, workspace=P, workspace_bytes=need - 1) == TOO_LARGE
    assert back(d_scale=P, workspace=P, workspace_bytes=need) == NULL
    assert back(linear_args(bias=P, scale=P), d_bias=P, d_scale=P, workspace=P, workspace_bytes=2 * need - 4) == TOO_LARGE
    assert back(dz=None) == 0                                    # nothing is wanted


def test_c_abi_refuses_products(lib):
    ok = dict(a=P, a_pitch=40, at=0, b=P, b_pitch=40, bt=0, type=1, out=P, M=64, N=32, K=40, workspace=None, bytes=0)
    call = lambda **more: lib.s3r_product(*{**ok, **more}.values(), None)
    assert call(a=None) == call(b=None) == call(out=None) == NULL
    assert call(M=0) == call(N=0) == call(K=0) == call(a_pitch=39) == call(at=1) == call(b_pitch=24) == SHAPE
    assert call(type=0) == UNSUPPORTED and call(a=P + 8) == call(b_pitch=44) == call(out=P + 1) == ALIGNMENT and call(K=1 << 31, a_pitch=1 << 31, b_pitch=1 << 31) == TOO_LARGE


def rope_args(**more):
    return RopeArgs(**{**dict(batch=1, tokens=4, heads=2, kv_heads=1, head_dim=64, type=1, table_type=0, axes=2, pairs=16, rows=8, stride_b=1024, stride_t=256, qkv=P,
                              pos=P, cos=P, sin=P, q=P, k=P, v=P, q_normed=1, k_normed=1), **more})


@pytest.mark.parametrize("more, code", [
    (dict(qkv=None), NULL), (dict(q=None), NULL), (dict(k=None), NULL), (dict(v=None), NULL), (dict(batch=0), SHAPE), (dict(tokens=-1), SHAPE), (dict(heads=0), SHAPE),
    (dict(kv_heads=0), SHAPE), (dict(head_dim=63), UNSUPPORTED), (dict(head_dim=258), UNSUPPORTED), (dict(head_dim=0), UNSUPPORTED), (dict(type=3), UNSUPPORTED),
    (dict(kind=2), UNSUPPORTED), (dict(q_normed=0, q_weight=P), SHAPE), (dict(k_normed=0, k_bias=P), SHAPE), (dict(q_weight=P, param_type=9), UNSUPPORTED),
    (dict(pos=None), SHAPE), (dict(cos=None), SHAPE), (dict(sin=None), SHAPE), (dict(rows=0), SHAPE), (dict(pairs=17), SHAPE), (dict(axes=-1), SHAPE), (dict(axes=3), SHAPE),
    (dict(table_type=4), UNSUPPORTED), (dict(qkv=P + 1), ALIGNMENT), (dict(q=P + 1), ALIGNMENT), (dict(cos=P + 2), ALIGNMENT), (dict(pos=P + 4), ALIGNMENT),
    (dict(q_weight=P + 2), ALIGNMENT), (dict(tokens=1 << 31), TOO_LARGE), (dict(heads=5000), TOO_LARGE), (dict(pairs=1 << 30, axes=2), SHAPE)])
def test_c_abi_refuses_qkv(lib, more, code):
    assert lib.s3r_qkv_norm_rope_fwd(C.byref(rope_args(**more)), None) == code


def test_c_abi_refuses_qkv_gradients(lib):
    need = lib.s3r_qkv_norm_rope_bwd_workspace_bytes(1, 4, 2, 1, 64)
    back = lambda f=rope_args(), **g: lib.s3r_qkv_norm_rope_bwd(C.byref(f), C.byref(RopeGrad(**{**dict(dq=P, dk=P, dv=P, d_qkv=P), **g})), None)
    assert need > 0 and lib.s3r_qkv_norm_rope_bwd_workspace_bytes(0, 4, 2, 1, 64) == 0
    assert back(d_qkv=None) == NULL and lib.s3r_qkv_norm_rope_bwd(C.byref(rope_args()), None, None) == NULL
    assert back(dk=P + 1) == ALIGNMENT and back(d_q_weight=P) == TOO_LARGE and back(d_q_weight=P, workspace=P, workspace_bytes=need - 1) == TOO_LARGE
    assert back(rope_args(q_normed=0), d_q_bias=P, workspace=P, workspace_bytes=need) == SHAPE
