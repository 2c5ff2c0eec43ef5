"""Refusals, shape functions and host logic of the operators around the attention: nothing here needs a GPU."""
import ctypes as C

import pytest
import torch

from speed3r_b200 import _lib, ops

BF16, F32 = torch.bfloat16, torch.float32


def meta(*shape, dtype=F32, grad=False):
    return torch.zeros(*shape, dtype=dtype, device="meta", requires_grad=grad)


def raises(text, call):
    with pytest.raises(RuntimeError, match=text):
        call()


def test_cpu_tensors_are_refused():
    x, w = torch.zeros(2, 4, 8), torch.ones(8)
    raises("no CPU path", lambda: ops.residual_norm(x, x, (w, w, 1e-5)))
    raises("no CPU path", lambda: ops.residual_norm_int8(x, x, (w, w, 1e-5)))
    raises("no CPU path", lambda: ops.quantize_tokens(x))
    q = torch.zeros(2, 8, dtype=torch.int8)
    raises("no CPU path", lambda: ops.int8_linear(q, torch.ones(2), q, torch.ones(2)))
    raises("no CPU path", lambda: ops.grad_norm([w]))
    raises("no CPU path", lambda: ops.adamw_step([w], [w], [w.clone()], [w.clone()], torch.zeros((), dtype=torch.int64)))
    raises("no CPU path", lambda: ops.adamw_state([w.byte()], [w.byte()], [torch.zeros(2, 1, dtype=torch.uint8)]))


@pytest.mark.parametrize("kw, text", [
    (dict(kind="batch"), "kind must be"),
    (dict(y=meta(2, 4, 9)), "not like x"),
    (dict(y=None, scale=meta(8)), "need a branch"),
    (dict(y=None, gate=meta(2, 1, 1)), "need a branch"),
    (dict(y=None, post_norm=(meta(8), None, 1e-5)), "need a branch"),
    (dict(y=None, norm=None), "nothing to compute"),
    (dict(gate=meta(2, 4, 8)), "gate must be"),
    (dict(gate=meta(2, 3, 1)), "gate must be"),
    (dict(gate=meta(8)), "as many dimensions"),
    (dict(gate=meta(3, 1, 1)), "gate of"),
    (dict(out_dtype=torch.float64), "out_dtype must be"),
])
def test_norm_refusals(kw, text):
    args = dict(y=meta(2, 4, 8), norm=(meta(8), meta(8), 1e-5))
    args.update(kw)
    raises(text, lambda: ops.residual_norm(meta(2, 4, 8), **args))


def test_norm_shapes_and_types():
    x, y, w = meta(2, 3, 4, 40, grad=True), meta(2, 3, 4, 40, dtype=BF16, grad=True), meta(40, dtype=BF16, grad=True)
    gate = meta(2, 1, 1, 40, grad=True)
    r, h = ops.residual_norm(x, y, (w, meta(40), 1e-5), scale=w, gate=gate, out_dtype=BF16)
    assert r.shape == h.shape == x.shape and r.dtype == F32 and h.dtype == BF16
    g = torch.autograd.grad((r, h), (x, y, w, gate), (r, h))
    assert [t.shape for t in g] == [x.shape, y.shape, w.shape, gate.shape] and [t.dtype for t in g] == [F32, BF16, BF16, F32]
    r, h = ops.residual_norm(x, None, (None, None, 1e-5))
    assert r is x and h.shape == x.shape and h.dtype == F32
    r, h = ops.residual_norm(x, y)
    assert h is None and r.shape == x.shape
    with torch.no_grad():
        r, q, s = ops.residual_norm_int8(x, y, (w, None, 1e-5))
    assert q.shape == x.shape and q.dtype == torch.int8 and s.shape == x.shape[:-1] and q.stride(-2) == 48


def test_what_has_no_gradient_says_so():
    x, w = meta(2, 4, 8, grad=True), meta(8)
    raises("forward-only", lambda: ops.residual_norm_int8(x, x, (w, None, 1e-5)))
    raises("forward-only", lambda: ops.quantize_tokens(x))
    q = meta(2, 8, dtype=torch.int8)
    raises("forward-only", lambda: ops.int8_linear(q, meta(2, grad=True), q, meta(2)))
    raises("needs a norm", lambda: ops.residual_norm_int8(meta(2, 4, 8)))
    r, h = ops.residual_norm(x, meta(2, 4, 8), (w, None, 1e-5))
    (g,) = torch.autograd.grad(h, x, h, create_graph=True)
    raises("cannot be differentiated again", lambda: torch.autograd.grad(g, x, g))
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(torch.zeros(2, 4, 8), torch.zeros(2, 4, 8))
        with pytest.raises(NotImplementedError):
            ops.residual_norm(dual, None, (torch.ones(8), None, 1e-5))


def test_linear_shapes():
    q, s = ops.quantize_tokens(meta(2, 3, 40))
    assert q.shape == (2, 3, 40) and s.shape == (2, 3)
    y = ops.int8_linear(q, s, meta(7, 40, dtype=torch.int8), meta(7))
    assert y.shape == (2, 3, 7) and y.dtype == BF16
    raises("out_dtype must be", lambda: ops.int8_linear(q, s, meta(7, 40, dtype=torch.int8), meta(7), out_dtype=torch.float64))


@pytest.mark.parametrize("kw, text", [(dict(seed=-1), "seed"), (dict(seed=1 << 63), "seed"), (dict(max_norm=0.0), "max_norm"), (dict(max_norm=1.0), "needs grad_norm")])
def test_adamw_refusals(kw, text):
    t = [meta(4)]
    raises(text, lambda: ops.adamw_step(t, t, t, t, torch.zeros((), dtype=torch.int64, device="meta"), **kw))


# ---- the C boundary ------------------------------------------------------------------------------------------------------
class NormArgs(C.Structure):
    _fields_ = ([("batch", C.c_int64), ("tokens", C.c_int64), ("channels", C.c_int), ("kind", C.c_int), ("post", C.c_int), ("eps", C.c_float),
                 ("post_eps", C.c_float)] + [(n, C.c_int) for n in ("x_type", "y_type", "h_type", "param_type", "gate_type", "gate_mode")] +
                [("gate_stride_b", C.c_int64), ("gate_stride_t", C.c_int64)] +
                [(n, C.c_void_p) for n in ("x", "y", "weight", "bias", "scale", "post_weight", "post_bias", "gate", "r", "h", "q", "q_scale")] +
                [("q_pitch", C.c_int64), ("stats", C.c_void_p)])


def test_norm_arguments_are_checked_without_a_gpu(lib):
    buf = C.create_string_buffer(4096)
    p = (C.addressof(buf) + 255) & ~255

    def rc(**kw):
        a = NormArgs(batch=1, tokens=2, channels=8, x=p, y=p, r=p, h=p)
        for k, v in kw.items():
            setattr(a, k, v)
        return lib.s3r_residual_norm_fwd(C.byref(a), None)

    assert lib.s3r_residual_norm_fwd(None, None) == -4
    assert rc(x=None) == -4 and rc(r=None) == -4 and rc(y=None, r=None, h=None) == -4
    assert rc(batch=0) == -1 and rc(tokens=-1) == -1 and rc(channels=0) == -1
    assert rc(channels=8193) == -6 and rc(batch=1 << 31) == -6
    assert rc(kind=2) == -2 and rc(x_type=3) == -2 and rc(gate_mode=3, gate=p) == -2
    assert rc(gate_mode=1) == -4 and rc(gate=p) == -4 and rc(y=None, scale=p) == -4
    assert rc(x=p + 1) == -3 and rc(weight=p + 2) == -3
    assert rc(q=p) == -2 and rc(h=None, q=p) == -1 and rc(h=None, q=p, q_scale=p, q_pitch=7) == -1
    assert lib.s3r_residual_norm_bwd(None, None, None) == -4
    assert lib.s3r_residual_norm_bwd_workspace_bytes(1, 100, 8, 0) > 0 and lib.s3r_residual_norm_bwd_workspace_bytes(0, 1, 8, 0) == 0


def test_int8_arguments_are_checked_without_a_gpu(lib):
    buf = C.create_string_buffer(4096)
    p = (C.addressof(buf) + 255) & ~255
    q = lambda x=p, type=0, xp=16, qq=p, qp=16, s=p, rows=1, ch=16: lib.s3r_quantize_rows(x, type, xp, qq, qp, s, rows, ch, None)
    assert q(x=None) == -4 and q(rows=0) == -1 and q(ch=17) == -1 and q(qp=8) == -1 and q(type=5) == -2 and q(x=p + 2) == -3 and q(rows=1 << 31) == -6
    f = lambda a=p, ap=32, b=p, bp=32, out=p, type=1, M=1, N=1, K=32: lib.s3r_int8_linear(a, ap, p, b, bp, p, None, out, type, M, N, K, None)
    assert f(a=None) == -4 and f(M=0) == -1 and f(K=33) == -1 and f(type=9) == -2 and f(ap=65552, bp=65552, K=65537) == -6
    r = lambda src=p + 1, sp=5, dst=p, dp=16, rows=3, K=5: lib.s3r_pad_rows(src, sp, dst, dp, rows, K, None)
    assert r(src=None) == -4 and r(rows=0) == -1 and r(dp=8, K=9) == -1 and r(dp=24) == -3 and r(dst=p + 8) == -3
    assert f(a=p + 1) == -3 and f(ap=40) == -3 and f(b=p + 8) == -3 and f(out=p + 1) == -3


class AdamArgs(C.Structure):
    _fields_ = [("n", C.c_int)] + [(n, C.c_void_p) for n in ("params", "grads", "m", "v", "m_exponents", "v_exponents", "counts", "param_types", "grad_types",
                                                             "step", "lr")] + \
               [(n, C.c_double) for n in ("lr_host", "beta1", "beta2", "eps", "weight_decay")] + [("norm", C.c_void_p), ("max_norm", C.c_double),
                                                                                                  ("seed", C.c_int64), ("workspace", C.c_void_p)]


def test_adamw_arguments_are_checked_without_a_gpu(lib):
    buf = C.create_string_buffer(4096)
    p = (C.addressof(buf) + 255) & ~255
    one = (C.c_void_p * 1)(p)
    odd = (C.c_void_p * 1)(p + 2)
    none = (C.c_void_p * 1)(None)
    count, types = (C.c_int64 * 1)(4), (C.c_int * 1)(0)
    at = lambda x: C.cast(x, C.c_void_p)

    def rc(**kw):
        a = AdamArgs(n=1, params=at(one), grads=at(one), m=at(one), v=at(one), counts=at(count), param_types=at(types), grad_types=at(types), step=p,
                     lr_host=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, seed=-1, workspace=p)
        for k, v in kw.items():
            setattr(a, k, v)
        return lib.s3r_adamw_step(C.byref(a), None)

    assert lib.s3r_adamw_step(None, None) == -4
    assert rc(n=-1) == -1 and rc(step=None) == -4 and rc(workspace=None) == -4 and rc(params=None) == -4 and rc(params=at(none)) == -4
    assert rc(beta1=1.0) == -2 and rc(eps=-1.0) == -2 and rc(params=at(odd)) == -3 and rc(m=at(odd)) == -3 and rc(step=p + 4) == -3
    assert rc(counts=at((C.c_int64 * 1)(-1))) == -1 and rc(param_types=at((C.c_int * 1)(3))) == -2 and rc(m_exponents=at(one)) == -4
    assert lib.s3r_grad_norm(1, None, None, None, p, p, 64, None) == -4
    assert lib.s3r_grad_norm(1, at(one), at(count), at(types), p, p, 0, None) == -6
    assert lib.s3r_adamw_state(1, at(none), at(one), at(one), at(one), at(one), at(one), at(count), None) == -4
