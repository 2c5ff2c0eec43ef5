"""The operators around the attention against plain 64-bit arithmetic: residual and norms, 8-bit tokens and products, AdamW.

Tolerances: a rounding to a type is off by at most eps / 2 of the value.  What is computed in fp32 in front of it adds a few times
2^-24 of the magnitudes that went into it; the factors below count those operations generously (sums of n terms by n)."""
import itertools
import math

import pytest
import torch

from speed3r_b200 import _lib, ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32 = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def close(got, want, dtype, fp32, what=""):
    """|got - want| within half a step of `dtype`, and `fp32` (a bound of the fp32 arithmetic in front, same shape or a number).
    Below a type's normal numbers the step is that of the smallest one."""
    assert got.dtype == dtype and got.shape == want.shape, f"{what}: {got.dtype} {tuple(got.shape)} for {dtype} {tuple(want.shape)}"
    allowed = half_step(dtype) * (want.abs() + fp32) + torch.finfo(dtype).tiny * half_step(dtype) * 2 + fp32
    off = (got.double() - want).abs()
    bad = ~(off <= allowed)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst by {(off - allowed)[bad].max().item():.3g} over the bound"


# ---- residual and norms ------------------------------------------------------------------------------------------------
def statistics(v, kind, eps):
    mean = v.mean(-1, keepdim=True) if kind == "layer" else torch.zeros_like(v[..., :1])
    return mean, 1 / torch.sqrt(((v - mean) ** 2).mean(-1, keepdim=True) + eps)


def through(d, n, inv, kind):
    flat = d.mean(-1, keepdim=True) if kind == "layer" else 0
    return inv * (d - flat - n * (d * n).mean(-1, keepdim=True))


class Norm:
    """One call's inputs, and its results in 64 bits (given the kernel's own r, whose rounding is checked by itself)."""

    def __init__(self, shape, x=torch.float32, y=torch.bfloat16, h=torch.bfloat16, w=torch.float32, kind="layer", affine=True, scale=True,
                 gate=None, post=False, branch=True, norm=True, seed=0, spread=1.0):
        g = torch.Generator(device=DEV).manual_seed(seed)
        rand = lambda *s: torch.randn(*s, device=DEV, generator=g)
        C = shape[-1]
        self.kind, self.h_type = kind, h
        self.x = (rand(*shape) * spread + 0.5).to(x)
        self.y = rand(*shape).to(y) if branch else None
        self.w = (1 + 0.3 * rand(C)).to(w) if affine and norm else None
        self.b = (0.3 * rand(C)).to(w) if affine and norm else None
        self.pw = (1 + 0.3 * rand(C)).to(w) if post else None
        self.pb = (0.3 * rand(C)).to(w) if post else None
        self.scale = (0.5 * rand(C)).to(w) if scale and branch else None
        self.gate = None if gate is None else (0.7 * rand(*gate)).to(w)
        self.norm = (self.w, self.b, 1e-5) if norm else None
        self.post = (self.pw, self.pb, 1e-6) if post else None
        self.dr, self.dh = rand(*shape).to(x), rand(*shape).to(h)

    def leaves(self):
        named = dict(x=self.x, y=self.y, w=self.w, b=self.b, scale=self.scale, gate=self.gate, pw=self.pw, pb=self.pb)
        return {n: t for n, t in named.items() if t is not None}

    def call(self):
        return ops.residual_norm(self.x, self.y, self.norm, self.scale, self.gate, self.post, self.kind, self.h_type)

    def check(self, r, h, grads=None):
        of = lambda t, other: torch.full((), float(other), dtype=torch.float64, device=DEV) if t is None else t.detach().double()
        x, C = self.x.detach().double(), self.x.shape[-1]
        c, gate, w, b, pw, pb = (of(*p) for p in ((self.scale, 1), (self.gate, 1), (self.w, 1), (self.b, 0), (self.pw, 1), (self.pb, 0)))
        tiny = 64 * F32
        if self.y is not None:
            y = self.y.detach().double()
            if self.post:
                mean, inv = statistics(y, self.kind, 1e-6)
                n = (y - mean) * inv
                u = n * pw + pb
            else:
                n, u = None, y
            branch = u * c * gate
            far = tiny * (u.abs().amax(-1, keepdim=True) * (c * gate).abs() if self.post else branch.abs())
            close(r, x + branch, self.x.dtype, far + 2 * F32 * x.abs(), "r")
        r64 = r.detach().double()
        G = self.dr.double() if self.y is not None else torch.zeros_like(x)
        if self.norm is not None:
            mean, inv = statistics(r64, self.kind, 1e-5)
            nr = (r64 - mean) * inv
            # the mean is off by a few 2^-24 of the row's magnitude, and with it every centred value
            row = r64.abs().amax(-1, keepdim=True) * inv
            far = tiny * ((row + nr.abs()) * w.abs() + b.abs())
            close(h, nr * w + b, self.h_type, far, "h")
        else:
            assert h is None
        if grads is None:
            return
        if self.norm is not None:
            dh = self.dh.double()
            d = dh * w
            G = G + through(d, nr, inv, self.kind)
            big = inv * d.abs().amax(-1, keepdim=True) * (1 + nr.abs()) * (1 + row)
            rows = lambda t: t.reshape(-1, C).sum(0)
            n_rows = x.numel() // C
            for name, term, err in (("w", dh * nr, dh.abs() * (row + nr.abs())), ("b", dh, dh.abs())):
                if name in grads:
                    close(grads[name], rows(term), self.w.dtype, (tiny + n_rows * F32) * rows(err), "d" + name)
        else:
            big = torch.zeros_like(G)
        g_far = tiny * (big + G.abs())
        close(grads["x"], G, self.x.dtype, g_far, "dx")
        if self.y is None:
            return
        du = G * c * gate
        du_far = g_far * (c * gate).abs() + tiny * du.abs()
        if self.post:
            e = du * pw
            dy = through(e, n, inv_y := statistics(y, self.kind, 1e-6)[1], self.kind)
            row_y = y.abs().amax(-1, keepdim=True) * inv_y
            dy_far = inv_y * (1 + n.abs()) * (1 + row_y) * (du_far * pw.abs() + tiny * e.abs()).amax(-1, keepdim=True) * 4
        else:
            dy, dy_far, row_y = du, du_far, 0
        if "y" in grads:
            close(grads["y"], dy, self.y.dtype, dy_far, "dy")
        n_rows = x.numel() // C

        def summed(name, term, err, dims, like):
            if name in grads:
                sums = lambda t: (t.sum(dims, keepdim=True) if dims else t).reshape(like.shape)
                count = term.numel() // like.numel()
                close(grads[name], sums(term), like.dtype, sums(err) + (tiny + count * F32) * sums(term.abs()), "d" + name)

        lead = tuple(range(x.dim() - 1))
        u_err = (tiny * u.abs().amax(-1, keepdim=True)) if self.post else 0
        one = torch.ones_like(x)
        if self.scale is not None:
            summed("scale", G * gate * u, (g_far * u.abs() + G.abs() * u_err) * gate.abs(), lead, self.scale)
        if self.gate is not None:
            over = tuple(i for i in range(x.dim()) if self.gate.shape[i] == 1 and x.shape[i] != 1)
            term = G * c * u * one
            summed("gate", term, (g_far * u.abs() + G.abs() * u_err) * c.abs() * one, over, self.gate)
        if self.post:
            summed("pw", du * n, du_far * n.abs() + du.abs() * tiny * (row_y + n.abs()), lead, self.pw)
            summed("pb", du, du_far, lead, self.pb)

    def train(self):
        leaves = self.leaves()
        for t in leaves.values():
            t.requires_grad_(True)
        r, h = self.call()
        outs = [(o, d) for o, d in ((r if self.y is not None else None, self.dr), (h, self.dh)) if o is not None]
        grads = dict(zip(leaves, torch.autograd.grad([o for o, _ in outs], list(leaves.values()), [d for _, d in outs])))
        self.check(r.detach(), None if h is None else h.detach(), grads)


@pytest.mark.parametrize("C", [1, 2, 7, 64, 100, 255, 256, 257, 511, 512, 768, 1000, 1023, 1024, 1028, 1540, 2048, 2049, 4096, 4100, 8191, 8192])
@pytest.mark.parametrize("kind", ["layer", "rms"])
def test_norm_widths(C, kind):
    Norm((2, 5, C), kind=kind, seed=C).train()


@pytest.mark.parametrize("rows", [(1, 1), (1, 2), (3, 1), (1, 300), (2, 701), (5, 1041)])
@pytest.mark.parametrize("post, gate", [(False, None), (True, "channel"), (True, "token"), (False, "sample")])
def test_norm_lengths_gates_and_post_norms(rows, post, gate):
    B, T = rows
    C = 192
    shape = {None: None, "channel": (B, 1, C), "token": (B, T, 1), "sample": (B, 1, 1)}[gate]
    Norm((B, T, C), post=post, gate=shape, seed=B + T).train()


@pytest.mark.parametrize("x, y, h, w", list(itertools.product([torch.float32, torch.bfloat16, torch.float16], [torch.float32, torch.bfloat16, torch.float16],
                                                               [torch.float32, torch.bfloat16, torch.float16], [torch.float32, torch.bfloat16])))
def test_norm_types(x, y, h, w):
    Norm((2, 9, 328), x=x, y=y, h=h, w=w, gate=(2, 1, 328), post=True, seed=3).train()
    Norm((2, 9, 131), x=x, y=y, h=h, w=w, gate=(2, 9, 1), seed=4).train()


@pytest.mark.parametrize("kw", [dict(branch=False), dict(norm=False), dict(affine=False), dict(scale=False), dict(norm=False, post=True, gate=(2, 1, 1)),
                                dict(gate=(1, 1, 260)), dict(gate=(1, 6, 1)), dict(gate=(1, 1, 1)), dict(gate=(2, 1, 260), scale=False, affine=False)])
def test_norm_parts_left_out(kw):
    Norm((2, 6, 260), seed=9, **kw).train()


@pytest.mark.parametrize("shape, gate", [((40,), None), ((7, 40), (7, 1)), ((2, 3, 4, 40), (2, 1, 1, 40)), ((2, 3, 4, 40), (1, 3, 4, 1)), ((2, 3, 1), (2, 3, 1))])
def test_norm_dimensions(shape, gate):
    Norm(shape, gate=gate, post=True, seed=5).train()


@pytest.mark.parametrize("C", [260, 500, 511, 512, 516, 700, 767, 768, 772, 1100, 1540])
@pytest.mark.parametrize("rows, x, post", [(3, torch.float32, False), (5003, torch.float32, True), (5003, torch.bfloat16, False)])
def test_norm_rows_of_three_six_and_two_warps(C, rows, x, post):
    n = Norm((1, rows, C), x=x, y=torch.bfloat16, post=post, seed=C, gate=(1, rows, 1))
    n.train()
    n.h_type = torch.float32
    with torch.no_grad():
        r, h = n.call()
        r8, q, s = ops.residual_norm_int8(n.x, n.y, n.norm, n.scale, n.gate, n.post, n.kind)
        q2, s2 = ops.quantize_tokens(h)
    assert torch.equal(r8, r) and torch.equal(q, q2) and torch.equal(s, s2)


def test_norm_training_size():
    Norm((2, 6144, 1024), gate=(2, 1, 1), seed=1).train()


def test_norm_strong_channels_and_offsets():
    """A mean a thousand times the spread: the variance comes from centred values."""
    n = Norm((1, 33, 512), x=torch.float32, h=torch.float32, spread=1.0, seed=2)
    n.x = n.x + 1000.0
    n.train()


def test_norm_only_one_gradient_arrives():
    n = Norm((2, 17, 320), seed=6, gate=(2, 17, 1))
    leaves = n.leaves()
    for t in leaves.values():
        t.requires_grad_(True)
    r, h = n.call()
    only_r = torch.autograd.grad(r, [n.x, n.y, n.scale, n.gate], n.dr, retain_graph=True)
    assert torch.equal(only_r[0], n.dr)
    close(only_r[1], n.dr.double() * n.scale.detach().double() * n.gate.detach().double(), n.y.dtype, 8 * F32 * n.dr.double().abs() * n.scale.detach().double().abs() * n.gate.detach().double().abs(), "dy")
    dx, dw = torch.autograd.grad(h, [n.x, n.w], n.dh)
    n.dr = torch.zeros_like(n.dr)
    n.check(r.detach(), h.detach(), {"x": dx, "w": dw})


def test_norm_of_constant_rows_and_values_that_are_not_finite():
    x = torch.full((1, 3, 256), 3.0, device=DEV)
    x[0, 1, 7], x[0, 2, 9] = math.inf, math.nan
    w = torch.ones(256, device=DEV)
    r, h = ops.residual_norm(x, torch.zeros_like(x), (w, None, 1e-5))
    assert torch.equal(h[0, 0], torch.zeros(256, device=DEV))
    assert h[0, 1:].isnan().all()
    assert torch.equal(r[0, 0], x[0, 0])
    _, q, s = ops.residual_norm_int8(x, None, (w, None, 1e-5))
    assert s[0, 0] == 0 and (q[0, 0] == 0).all() and s[0, 1:].isnan().all()


def test_norm_gradients_against_differences():
    g = torch.Generator(device=DEV).manual_seed(0)
    n = Norm((2, 3, 24), x=torch.float32, y=torch.float32, h=torch.float32, gate=(2, 1, 24), post=True, seed=8)
    leaves = n.leaves()
    for t in leaves.values():
        t.requires_grad_(True)
    r, h = n.call()
    loss = lambda r, h: (r.double() * n.dr.double()).sum() + (h.double() * n.dh.double()).sum()
    grads = torch.autograd.grad(loss(r, h), list(leaves.values()))
    step = 2.0 ** -7
    for (name, t), grad in zip(leaves.items(), grads):
        way = torch.randn(t.shape, device=DEV, generator=g)
        with torch.no_grad():
            keep = t.clone()
            t.copy_(keep + step * way)
            up = loss(*n.call())
            t.copy_(keep - step * way)
            down = loss(*n.call())
            t.copy_(keep)
        want, got = ((up - down) / (2 * step)).item(), (grad.double() * way.double()).sum().item()
        # central differences: third derivatives x step^2 (6e-5), and the loss's rounding (144 terms x 2^-22) over the step
        size = (grad.double().norm() * way.double().norm()).item()
        assert abs(got - want) <= 1e-2 * size + 1e-2, (name, got, want)


@pytest.mark.parametrize("C, rows", [(16, 3), (100, 5), (1000, 40), (1024, 1), (1024, 700), (1027, 9), (4096, 3), (8192, 2)])
def test_norm_int8_is_the_quantised_norm(C, rows):
    n = Norm((1, rows, C), h=torch.float32, seed=C + rows, gate=(1, rows, 1))
    r, h = n.call()
    r8, q, s = ops.residual_norm_int8(n.x, n.y, n.norm, n.scale, n.gate, n.post, n.kind)
    assert torch.equal(r8, r) and q.dtype == torch.int8 and q.shape == n.x.shape and s.shape == (1, rows) and (rows == 1 or q.stride(-2) % 16 == 0)
    q2, s2 = ops.quantize_tokens(h)
    assert torch.equal(q, q2) and torch.equal(s, s2)


def test_norm_strides_and_addresses():
    """Transposed and sliced tensors, and views that begin anywhere."""
    base = torch.randn(2, 320, 12, device=DEV).transpose(1, 2)
    y = torch.randn(2, 12, 640, device=DEV)[..., 1:321]
    w = torch.randn(321, device=DEV)[1:]
    r, h = ops.residual_norm(base, y, (w, None, 1e-5), kind="rms")
    r2, h2 = ops.residual_norm(base.contiguous(), y.contiguous(), (w.clone(), None, 1e-5), kind="rms")
    assert torch.equal(r, r2)
    close(h, h2.double(), torch.float32, 64 * F32 * h2.double().abs(), "h")
    flat = torch.randn(2 * 12 * 320 + 1, device=DEV)
    one = flat[1:].view(2, 12, 320)
    r, h = ops.residual_norm(one, y, (w, None, 1e-5))
    r2, h2 = ops.residual_norm(one.clone(), y, (w, None, 1e-5))
    assert torch.equal(r, r2)
    close(h, h2.double(), torch.float32, 64 * F32 * (1 + h2.double().abs()), "h")


def test_norm_sums_do_not_depend_on_the_run():
    n = Norm((3, 997, 1024), gate=(3, 1, 1024), post=True, seed=12)
    leaves = n.leaves()
    for t in leaves.values():
        t.requires_grad_(True)
    first = torch.autograd.grad(n.call(), list(leaves.values()), (n.dr, n.dh))
    for _ in range(3):
        again = torch.autograd.grad(n.call(), list(leaves.values()), (n.dr, n.dh))
        assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_norm_without_rows():
    x = torch.zeros(2, 0, 64, device=DEV, requires_grad=True)
    w = torch.ones(64, device=DEV, requires_grad=True)
    r, h = ops.residual_norm(x, torch.zeros_like(x), (w, None, 1e-5), scale=w)
    assert r.shape == h.shape == x.shape
    gx, gw = torch.autograd.grad((r, h), (x, w), (torch.zeros_like(r), torch.zeros_like(h)))
    assert gx.shape == x.shape and (gw == 0).all()


# ---- 8 bits --------------------------------------------------------------------------------------------------------------
def quantised(x):
    big = x.float().abs().amax(-1)
    q = torch.where(big[..., None] > 0, x.float() * (127 / big)[..., None], 0).round()        # 127 / big: big's reciprocal, times 127
    return q.to(torch.int8), big / torch.full_like(big, 127)                                  # by a tensor: PyTorch multiplies by 1 / 127


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", [(1, 1), (3, 2), (2, 5, 17), (1, 1024), (400, 1024), (700, 255), (9, 1000), (5, 4096), (3, 4100), (2, 16384), (2, 16388), (3, 33001)])
def test_quantize_tokens(shape, dtype):
    x = torch.randn(*shape, device=DEV).to(dtype)
    x[..., 0, :] *= 100
    q, s = ops.quantize_tokens(x)
    want, scale = quantised(x)
    assert torch.equal(q, want) and torch.equal(s, scale)
    assert x.numel() == x.shape[-1] or q.stride(-2) % 16 == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows", [1, 297, 501])
@pytest.mark.parametrize("C", [256, 260, 509, 512, 1023, 1028, 1536, 2047, 2048, 2052])
def test_quantize_tokens_of_few_and_many_rows(rows, C, dtype):
    x = torch.randn(rows, C, device=DEV, generator=torch.Generator(device=DEV).manual_seed(C)).to(dtype)
    x[rows // 2, C - 1] = 50.0
    q, s = ops.quantize_tokens(x)
    want, scale = quantised(x)
    assert torch.equal(q, want) and torch.equal(s, scale)


def test_quantize_tokens_rows_of_a_slice_zeros_and_values_that_are_not_finite():
    x = torch.randn(50, 640, device=DEV)
    for part in (x[:, 3:200], x[::2, :320], x.t(), x[:1, 1:100]):
        q, s = ops.quantize_tokens(part)
        want, scale = quantised(part)
        assert torch.equal(q, want) and torch.equal(s, scale)
    x = torch.zeros(4, 64, device=DEV)
    x[1, 3], x[2, 5], x[3, 1] = math.nan, math.inf, 1e-40
    q, s = ops.quantize_tokens(x)
    assert (q[0] == 0).all() and s[0] == 0 and s[1].isnan() and s[2].isinf() and (q[3] == 0).all()


def linear_reference(q, s, w, ws, bias):
    y = (q.double() @ w.double().T) * s.double().unsqueeze(-1) * ws.double()
    return y if bias is None else y + bias.double()


def int8(*shape, lo=-127, hi=128):
    return torch.randint(lo, hi, shape, device=DEV, dtype=torch.int8)


def check_linear(M, N, K, dtype=torch.bfloat16, bias=True, lead=None):
    q, w = int8(M, K), int8(N, K)
    s, ws = torch.rand(M, device=DEV) + 0.1, torch.rand(N, device=DEV) * 0.01
    b = torch.randn(N, device=DEV) if bias else None
    if lead:
        q, s = q.view(*lead, K), s.view(lead)
    got = ops.int8_linear(q, s, w, ws, b, dtype)
    want = linear_reference(q, s, w, ws, b)
    # the sum's conversion, two products and a sum
    close(got, want, dtype, 4 * F32 * (want.abs() + 2 * (0 if b is None else b.abs().double())), f"{M} x {N} x {K}")


@pytest.mark.parametrize("K", [1, 3, 16, 31, 32, 100, 128, 129, 255, 256, 1000, 1024, 4096])
@pytest.mark.parametrize("M, N", [(1, 1), (1, 64), (1, 1000), (2, 333), (16, 256), (17, 48), (33, 129), (64, 65), (65, 8), (128, 256), (129, 257), (500, 1000)])
def test_int8_linear_sizes(M, N, K):
    check_linear(M, N, K)


@pytest.mark.parametrize("M", [1, 2, 3, 4, 5, 8, 9])
@pytest.mark.parametrize("N, K", [(1, 5), (31, 16), (33, 500), (1000, 1040), (4096, 1024), (129, 6000), (129, 6160), (40, 50000)])
def test_int8_linear_few_tokens(M, N, K):
    check_linear(M, N, K, torch.float32 if N % 2 else torch.bfloat16)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M, N, K", [(1, 1024, 1024), (8, 4096, 1024), (100, 1000, 500), (300, 3104, 1024), (2048, 1024, 4096), (8328, 3104, 1024), (4001, 1023, 700), (20000, 512, 256)])
@pytest.mark.parametrize("bias", [True, False])
def test_int8_linear_types(M, N, K, dtype, bias):
    check_linear(M, N, K, dtype, bias)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N", [1, 5, 7, 9, 63, 65, 67, 129, 250, 261, 517])
@pytest.mark.parametrize("start", [0, 1, 2, 3, 5])
def test_int8_linear_results_that_begin_anywhere(N, start, dtype):
    """Through the library's C entry, into the middle of a buffer: what is around the result stays."""
    M, K = 301, 144
    q, w = int8(M, K), int8(N, K)
    s, ws = torch.rand(M, device=DEV) + 0.5, torch.rand(N, device=DEV) + 0.5
    whole = torch.full((start + M * N + 40,), 7.0, device=DEV, dtype=dtype)
    code = {torch.float32: 0, torch.bfloat16: 1}[dtype]
    rc = _lib.load().s3r_int8_linear(q.data_ptr(), K, s.data_ptr(), w.data_ptr(), K, ws.data_ptr(), None, whole.data_ptr() + start * whole.element_size(), code, M, N, K,
                               torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    assert torch.equal(whole[start:start + M * N].view(M, N), ops.int8_linear(q, s, w, ws, None, dtype))
    assert (whole[:start] == 7).all() and (whole[start + M * N:] == 7).all()


def test_int8_linear_largest_sums_are_exact():
    """Sums near 2^31: 65536 products of 127 x 127 would be 2^30; with -128 on both sides they are 2^30."""
    for M in (1, 5, 200):
        K, N = 65536, 40
        q, w = torch.full((M, K), -128, device=DEV, dtype=torch.int8), torch.full((N, K), -128, device=DEV, dtype=torch.int8)
        w[1] = 127
        got = ops.int8_linear(q, torch.ones(M, device=DEV), w, torch.ones(N, device=DEV), None, torch.float32)
        assert (got[:, 0] == 2.0 ** 30).all()
        assert (got[:, 1] == float(torch.tensor(-128 * 127 * K, dtype=torch.float32))).all()


def test_int8_linear_shapes_pitches_and_addresses():
    check_linear(24, 72, 96, lead=(2, 3, 4))
    check_linear(1, 72, 40, lead=())
    whole = int8(40, 1040)
    w = int8(72, 1040)
    s, ws = torch.ones(40, device=DEV), torch.ones(72, device=DEV)
    for a, b in ((whole[:, 16:816], w[:, 16:816]), (whole[:, 3:803], w[:, 5:805]), (whole[::2, :800], w[:, :800]), (whole[:1, :333], w[:, 7:340]),
                 (whole[:, 16:817], w[:, 32:833])):
        got = ops.int8_linear(a, s[: a.shape[0]], b, ws, None, torch.float32)
        assert torch.equal(got, (a.double() @ b.double().T).float())
    assert ops.int8_linear(whole[:0], s[:0], w, ws).shape == (0, 72)


@pytest.mark.parametrize("K", [1, 5, 16, 17, 31, 33, 1001, 4095])
def test_int8_linear_operands_that_begin_anywhere(K):
    """Tight rows of odd length, at any byte of a buffer: nothing in front of them or behind them is read."""
    for start in (0, 1, 2, 3, 5):
        flat_a, flat_b = int8(start + 20 * K), int8(start + 37 * K)
        a, b = flat_a[start:].view(20, K), flat_b[start:].view(37, K)
        for m in (20, 3):
            got = ops.int8_linear(a[:m], torch.ones(m, device=DEV), b, torch.ones(37, device=DEV), None, torch.float32)
            assert torch.equal(got, (a[:m].double() @ b.double().T).float())


def test_int8_linear_rows_of_scales_that_are_not_finite():
    q, w = int8(9, 64), int8(16, 64)
    s, ws = torch.ones(9, device=DEV), torch.ones(16, device=DEV)
    s[4] = math.nan
    y = ops.int8_linear(q, s, w, ws, None, torch.float32)
    assert y[4].isnan().all() and y[[0, 1, 2, 3, 5, 6, 7, 8]].isfinite().all()


# ---- AdamW ---------------------------------------------------------------------------------------------------------------
def philox(a, c, key):
    a, c = a.clone(), c.clone()
    for i in range(7):
        low, high = (a & 0xFFFF) * 0xD256D193, (a >> 16) * 0xD256D193
        whole_low, whole_high = (low + ((high & 0xFFFF) << 16)) & 0xFFFFFFFF, (high + (low >> 16)) >> 16
        a, c = (whole_high & 0xFFFFFFFF) ^ ((key + i * 0x9E3779B9) & 0xFFFFFFFF) ^ c, whole_low
    return torch.stack((a, c), -1).view(-1)


def values(code, e, bits):
    """64-bit meaning of codes with `bits` bits of exponent."""
    n = code.numel()
    code = torch.nn.functional.pad(code.reshape(-1), (0, -n % 256)).long().view(-1, 256)
    sign = 1.0 - 2.0 * ((code > 127) & (bits == 4))
    code = code % (8 << bits)
    E, f, top = code // 8, (code % 8).double() / 8, 2 ** bits - 1
    v = torch.where(E > 0, (1 + f) * torch.exp2((E - top).double()), f * 2.0 ** (1 - top))
    return (sign * v * torch.exp2(e.double() - 127)[:, None]).view(-1)[:n]


def grid_below(z, bits):
    """The step of the codes' grid at magnitude z (in units of the block's power of two)."""
    bottom = 2 - 2 ** bits
    return torch.exp2(torch.floor(torch.log2(z.clamp(min=2.0 ** -60))).clamp(min=bottom) - 3)


class Adam:
    def __init__(self, shapes, p=torch.float32, g=None, eight=False, seed=0):
        gen = torch.Generator(device=DEV).manual_seed(seed)
        rand = lambda s: torch.randn(s, device=DEV, generator=gen)
        self.eight = eight
        self.params = [rand(s).to(p) for s in shapes]
        self.step = torch.zeros((), dtype=torch.int64, device=DEV)
        self.gen, self.g = gen, g or p
        if eight:
            self.m = [torch.zeros(s, device=DEV, dtype=torch.uint8) for s in shapes]
            self.v = [torch.zeros(s, device=DEV, dtype=torch.uint8) for s in shapes]
            self.scales = [torch.full((2, -(-math.prod(s) // 256)), 27, device=DEV, dtype=torch.uint8) for s in shapes]
        else:
            self.m, self.v = [torch.zeros(s, device=DEV) for s in shapes], [torch.zeros(s, device=DEV) for s in shapes]
            self.scales = None
        self.fresh()

    def fresh(self):
        self.grads = [(torch.randn(p.shape, device=DEV, generator=self.gen) * torch.exp(torch.randn(p.shape, device=DEV, generator=self.gen))).to(self.g) for p in self.params]

    def states(self, i):
        if self.eight:
            return values(self.m[i], self.scales[i][0], 4), values(self.v[i], self.scales[i][1], 5)
        return self.m[i].double().view(-1), self.v[i].double().view(-1)

    def advance(self, lr=1e-2, b1=0.9, b2=0.99, eps=1e-8, decay=0.1, max_norm=None, seed=None):
        """One step, checked against the formula in 64 bits."""
        before = [(p.double().view(-1), *self.states(i)) for i, p in enumerate(self.params)]
        norm = ops.grad_norm(self.grads) if max_norm is not None else None
        factor = 1.0
        if norm is not None:
            exact = math.sqrt(sum((g.double() ** 2).sum().item() for g in self.grads))
            assert abs(norm.item() - exact) <= F32 * exact * 1.01
            factor = min(1.0, max_norm / (exact + 1e-6))
        t = int(self.step) + 1
        ops.adamw_step(self.params, self.grads, self.m, self.v, self.step, lr=lr, betas=(b1, b2), eps=eps, weight_decay=decay, grad_norm=norm,
                       max_norm=max_norm, scales=self.scales, seed=seed)
        assert int(self.step) == t
        for i, (p, m, v) in enumerate(before):
            g = self.grads[i].double().view(-1) * factor
            m1, v1 = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
            size = (b1 * m).abs() + ((1 - b1) * g).abs()
            root = torch.sqrt(v1 / (1 - b2 ** t)) + eps
            want = p * (1 - lr * decay) - lr / (1 - b1 ** t) * m1 / root
            got = self.params[i]
            # m, v, the root and the quotient: 2^-24 each, a few of them
            far = 8 * F32 * p.abs() + 40 * F32 * lr / (1 - b1 ** t) * size / root
            if seed is not None and got.dtype == torch.bfloat16:
                assert ((got.double().view(-1) - want).abs() <= 2 * half_step(got.dtype) * (want.abs() + far) * 2 + far).all()
            else:
                close(got.view(-1), want, got.dtype, far, f"p[{i}]")
            gm, gv = self.states(i)
            if not self.eight:
                assert ((gm - m1).abs() <= 4 * F32 * size + 1e-45).all() and ((gv - v1).abs() <= 6 * F32 * v1 + 1e-44).all()
                continue
            n = p.numel()
            low = None
            if seed is not None:
                pair = torch.arange((n + 1) // 2, device=DEV)
                low = philox(pair, torch.full_like(pair, t), (seed + i * 0x85EBCA6B) & 0xFFFFFFFF)[:n]
            for name, x, y, e, bits, random, width in (("m", m1, gm, self.scales[i][0], 4, None if low is None else low & 0xFF, 8),
                                                       ("v", v1, gv, self.scales[i][1], 5, None if low is None else low >> 8 & 0x3FFF, 14)):
                unit = torch.exp2(e.double() - 127).repeat_interleave(256)[:n]
                blocks = torch.nn.functional.pad(x.abs(), (0, -n % 256)).view(-1, 256).amax(1)
                top = 1.875 * torch.exp2(e.double() - 127)
                # the block's largest magnitude is within the codes, and would not be within those of half the unit
                assert (blocks <= top * (1 + 16 * F32)).all() and ((blocks > top / 2 * (1 - 16 * F32)) | (e == 27)).all(), name
                z = x.abs() / unit
                last = grid_below(z, bits)
                slack = 16 * F32 * (size / unit if name == "m" else z) + 2.0 ** -37
                if random is None:
                    off = (y.abs() / unit - z.clamp(max=1.875)).abs()
                    ok = off <= last / 2 + slack
                    if name == "v":
                        ok |= (y / unit - 2.0 ** -33).abs() < 2.0 ** -40          # never down to zero
                else:
                    where = z / last + (random.double() + 0.5) / 2 ** width
                    want = torch.floor(where) * last
                    near = (where - torch.round(where)).abs() * last <= slack      # fp32 may see the other side of a border
                    want = want.clamp(max=1.875)
                    if name == "v":
                        want = torch.where(z > 0, want.clamp(min=2.0 ** -33), want)
                    ok = (y.abs() / unit == want) | near
                    assert near.sum() <= 2 + 0.01 * n                              # few are
                assert ok.all(), f"{name}[{i}]: {int((~ok).sum())} of {n}"
                assert ((torch.sign(y) == torch.sign(x)) | (y == 0)).all()


SHAPES = [(1,), (3, 5), (255,), (256,), (257,), (64, 64), (1041, 33), (2048,), (5000,), (8, 3, 100)]


@pytest.mark.parametrize("p, g", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.float32, torch.bfloat16), (torch.float16, torch.float32)])
@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("seed", [None, 77])
def test_adamw_steps(p, g, eight, seed):
    a = Adam(SHAPES, p, g, eight, seed=1)
    for i in range(4):
        a.advance(max_norm=None if i < 2 else 1.0, seed=seed)
        a.fresh()


def test_adamw_many_tensors():
    a = Adam([(17 + i % 900,) for i in range(700)], eight=True)
    a.advance(seed=5, max_norm=1.0)
    a.fresh()
    a.advance(seed=5, max_norm=1e9)


@pytest.mark.parametrize("eight", [False, True])
def test_adamw_views_of_one_buffer(eight):
    """Tensors that begin anywhere in a buffer, next to what must not change."""
    a, b = Adam([(300,), (1000,), (4097,)], eight=eight, seed=3), Adam([(300,), (1000,), (4097,)], eight=eight, seed=3)
    guard = 3

    def moved(ts):
        flat = torch.full((sum(t.numel() + guard for t in ts),), 9, device=DEV).to(ts[0].dtype)
        views, at = [], 0
        for t in ts:
            at += guard
            flat[at:at + t.numel()] = t.reshape(-1)
            views.append(flat[at:at + t.numel()].view(t.shape))
            at += t.numel()
        return flat, views

    (fp, b.params), (_, b.grads), (fm, b.m), (fv, b.v) = moved(b.params), moved(b.grads), moved(b.m), moved(b.v)
    a.advance(seed=1 if eight else None)
    b.advance(seed=1 if eight else None)
    for x, y in itertools.chain(zip(a.params, b.params), zip(a.m, b.m), zip(a.v, b.v)):
        assert torch.equal(x, y)
    for flat in (fp, fm, fv):
        at = 0
        for t in a.params:
            assert (flat[at:at + guard] == 9).all()
            at += guard + t.numel()


def test_adamw_leaves_everything_where_the_norm_is_not_finite():
    for eight in (False, True):
        a = Adam([(1000,), (300,)], eight=eight)
        a.advance()
        kept = [t.clone() for t in a.params + a.m + a.v]
        a.grads[1][7] = math.inf
        norm = ops.grad_norm(a.grads)
        ops.adamw_step(a.params, a.grads, a.m, a.v, a.step, grad_norm=norm, max_norm=1.0, scales=a.scales)
        ops.adamw_step(a.params, a.grads, a.m, a.v, a.step, grad_norm=norm, scales=a.scales)
        assert int(a.step) == 1 and all(torch.equal(x, y) for x, y in zip(kept, a.params + a.m + a.v))


def test_adamw_gradients_that_are_not_finite_without_a_norm():
    """The block's state becomes NaN, its neighbours do not."""
    a = Adam([(1024,)], eight=True)
    a.grads[0][300] = math.nan
    ops.adamw_step(a.params, a.grads, a.m, a.v, a.step, scales=a.scales)
    m, v = ops.adamw_state(a.m, a.v, a.scales)
    assert m[0][256:512].isnan().all() and v[0][256:512].isnan().all() and a.params[0][300].isnan()
    rest = torch.cat((torch.arange(256), torch.arange(512, 1024))).to(DEV)
    assert m[0][rest].isfinite().all() and v[0][rest].isfinite().all() and int(a.params[0].isnan().sum()) == 1


def test_adamw_state_is_what_codes_stand_for():
    codes = torch.arange(256, device=DEV, dtype=torch.uint8).repeat(3)[:700].contiguous()
    e = torch.tensor([[27, 127, 200], [100, 255, 130]], device=DEV, dtype=torch.uint8)
    (m,), (v,) = ops.adamw_state([codes], [codes], [e])
    assert torch.equal(m.double(), values(codes, e[0], 4))
    want = values(codes, e[1], 5)
    want[256:512] = math.nan
    assert torch.equal(v.double().nan_to_num(7), want.nan_to_num(7)) and v[256:512].isnan().all()
    whole = torch.zeros(701, device=DEV), torch.zeros(701, device=DEV)
    ops.adamw_state([codes], [codes], [e], out=([whole[0][1:]], [whole[1][1:]]))
    assert torch.equal(whole[0][1:], m) and whole[0][0] == 0


@pytest.mark.parametrize("off", [0, 4, 1])
def test_adamw_state_of_outputs_that_begin_anywhere(off):
    """At a multiple of 32 bytes, of 16 and of neither; what is around them stays."""
    n = 5000
    codes = torch.randint(0, 256, (n,), device=DEV, dtype=torch.uint8)
    e = torch.randint(90, 160, (2, -(-n // 256)), device=DEV, dtype=torch.uint8)
    whole = torch.full((2, n + 9), 3.0, device=DEV)
    m, v = whole[0][off:off + n], torch.full((n + 9,), 3.0, device=DEV)[off:off + n]
    ops.adamw_state([codes], [codes], [e], out=([m], [v]))
    assert torch.equal(m.double(), values(codes, e[0], 4)) and torch.equal(v.double(), values(codes, e[1], 5))
    assert (whole[0][:off] == 3).all() and (whole[0][off + n:] == 3).all()


@pytest.mark.parametrize("sizes", [[1, 2_000_000, 5, 256, 257, 900_000, 3], [7, 300_000, 1] * 9, [40_000, 1, 513, 90_000, 2, 2, 1025, 600_000] * 50],
                         ids=["7", "27", "400"])
@pytest.mark.parametrize("eight", [False, True])
def test_adamw_finds_every_tensor(sizes, eight):
    """All in one call and one by one: bit for bit the same."""
    gen = torch.Generator(device=DEV).manual_seed(len(sizes))
    p, g = ([torch.randn(n, device=DEV, generator=gen) for n in sizes] for _ in range(2))
    m, v = ([torch.randint(0, 127, (n,), device=DEV, dtype=torch.uint8, generator=gen) if eight else torch.rand(n, device=DEV, generator=gen) for n in sizes]
            for _ in range(2))
    e = [torch.randint(110, 130, (2, -(-n // 256)), device=DEV, dtype=torch.uint8, generator=gen) for n in sizes] if eight else None
    all_at_once = [[t.clone() for t in x] if x else None for x in (p, m, v, e)]
    step = torch.zeros((), dtype=torch.int64, device=DEV)
    ops.adamw_step(all_at_once[0], g, all_at_once[1], all_at_once[2], step, scales=all_at_once[3])
    for i in range(len(sizes)):
        step.zero_()
        ops.adamw_step([p[i]], [g[i]], [m[i]], [v[i]], step, scales=[e[i]] if eight else None)
    for x, y in zip((p, m, v, e), all_at_once):
        assert x is None or all(torch.equal(a, b) for a, b in zip(x, y))
    want = sum((t.double() ** 2).sum() for t in g).sqrt()
    assert abs(ops.grad_norm(g).double() - want) <= 2.0 ** -23 * want
    if eight:
        for out, codes, k, bits in zip(ops.adamw_state(m, v, e), (m, v), (0, 1), (4, 5)):
            assert all(torch.equal(o.double(), values(c, s[k], bits)) for o, c, s in zip(out, codes, e))


def test_adamw_lr_on_the_device_and_mixed_states():
    a, b = Adam([(5000,), (10,)], seed=2), Adam([(5000,), (10,)], seed=2)
    ops.adamw_step(a.params, a.grads, a.m, a.v, a.step, lr=0.03)
    ops.adamw_step(b.params, b.grads, b.m, b.v, b.step, lr=torch.tensor(0.03, device=DEV))
    # 0.03 in 64 and in 32 bits
    assert all(((x - y).abs() <= 8 * F32 * x.abs() + 1e-8).all() for x, y in zip(a.params, b.params))
    c = Adam([(5000,), (10,)], eight=True, seed=2)
    c.m[1], c.v[1], c.scales[1] = torch.zeros(10, device=DEV), torch.zeros(10, device=DEV), None
    ops.adamw_step(c.params, c.grads, c.m, c.v, c.step, lr=0.03, scales=c.scales)
    assert torch.equal(c.m[1], a.m[1]) and torch.equal(c.params[1], a.params[1])


def test_adamw_stochastic_rounding_keeps_small_changes():
    """A second moment that shrinks by a thousandth a step: to nearest its codes stand still, stochastically they follow on average."""
    n, steps = 4096, 200
    got = {}
    for seed in (None, 3):
        v = torch.full((n,), 200, device=DEV, dtype=torch.uint8)
        v[::256] = 255                                  # the block's largest, kept up by its gradient
        m, e = torch.zeros(n, device=DEV, dtype=torch.uint8), torch.full((2, n // 256), 127, device=DEV, dtype=torch.uint8)
        g = torch.zeros(n, device=DEV)
        g[::256] = math.sqrt(1.875)
        p, step = torch.zeros(n, device=DEV), torch.zeros((), dtype=torch.int64, device=DEV)
        start = values(v, e[1], 5)[1].item()
        for _ in range(steps):
            ops.adamw_step([p], [g], [m], [v], step, lr=0.0, scales=[e], seed=seed)
        rest = torch.ones(n, dtype=torch.bool, device=DEV)
        rest[::256] = False
        got[seed] = values(v, e[1], 5)[rest].mean().item() / start
    assert got[None] == 1.0
    # 4080 elements whose random walk has a variance of about 200 x 0.001 x 0.125 of the value squared: 0.16 / sqrt(4080) = 0.0025
    assert abs(got[3] - 0.999 ** steps) < 5 * 0.0025


def test_grad_norm_sizes():
    for counts in ([1], [0, 5], [16384], [16385, 3, 0, 99999], [7] * 700):
        ts = [torch.randn(c, device=DEV).to([torch.float32, torch.bfloat16, torch.float16][i % 3]) for i, c in enumerate(counts)]
        want = math.sqrt(sum((t.double() ** 2).sum().item() for t in ts))
        assert abs(ops.grad_norm(ts).item() - want) <= F32 * want * 1.01
    big = torch.full((1 << 20,), 1e30, device=DEV)
    assert abs(ops.grad_norm([big]).item() - 1e30 * 1024) <= 1e-6 * 1e33
    flat = torch.randn(1000, device=DEV)
    assert abs(ops.grad_norm([flat[1:], flat.view(10, 100).t()]).item() - math.sqrt((flat[1:].double() ** 2).sum() + (flat.double() ** 2).sum())) < 1e-4


def test_norm_sums_are_the_same_for_few_rows_and_many():
    """r is rounded product by product, whichever kernel computes it."""
    n = Norm((1, 20000, 1024), gate=(1, 20000, 1), seed=3)
    r, _ = n.call()
    assert torch.equal(r, n.x + n.y.float() * n.scale * n.gate)
    n.x, n.y, n.gate = n.x[:, :50].contiguous(), n.y[:, :50].contiguous(), n.gate[:, :50].contiguous()
    assert torch.equal(n.call()[0], r[:, :50])


def test_adamw_codes_are_those_of_separate_operations():
    """Products and sums of the states are rounded one by one: codes are the same bits as PyTorch's operations give."""
    gen = torch.Generator(device=DEV).manual_seed(5)
    n = 1 << 22
    g = torch.randn(n, device=DEV, generator=gen) * torch.exp(2 * torch.randn(n, device=DEV, generator=gen))
    m, v = torch.randint(0, 256, (2, n), device=DEV, generator=gen, dtype=torch.uint8)
    e = torch.randint(110, 130, (2, n // 256), device=DEV, generator=gen, dtype=torch.uint8)
    m0, v0 = values(m, e[0], 4).float(), values(v, e[1], 5).float()
    m1, v1 = m0 * 0.9 + g * (1 - 0.9), v0 * 0.999 + g * g * (1 - 0.999)
    p, step = torch.zeros(n, device=DEV), torch.zeros((), dtype=torch.int64, device=DEV)
    m32, v32, step32 = m0.clone(), v0.clone(), step.clone()
    ops.adamw_step([p.clone()], [g], [m32], [v32], step32)
    assert torch.equal(m32, m1) and torch.equal(v32, v1)
    ops.adamw_step([p], [g], [m], [v], step, scales=[e])
    for x, code, exponent, bits in ((m1, m, e[0], 4), (v1, v, e[1], 5)):
        unit = torch.exp2(exponent.double() - 127).repeat_interleave(256)
        z = x.double().abs() / unit
        last = grid_below(z, bits)
        want = (torch.round(z / last) * last).clamp(max=1.875)
        want = torch.where(x > 0, want.clamp(min=2.0 ** -33), want) if bits == 5 else want
        assert torch.equal(values(code, exponent, bits).abs() / unit, want)


def test_norm_keeps_no_branch_that_nothing_multiplies():
    """Where neither scale nor gate is learnt the branch is not saved, and its gradient comes without it."""
    n = Norm((2, 333, 512), y=torch.bfloat16, gate=(2, 1, 1), seed=13)
    x, y = n.x.requires_grad_(True), n.y.requires_grad_(True)
    torch.cuda.synchronize()
    r, h = n.call()
    dx, dy = torch.autograd.grad((r, h), (x, y), (n.dr, n.dh))
    assert dy.dtype == torch.bfloat16
    n.check(r.detach(), h.detach(), dict(x=dx, y=dy))


def test_norm_beyond_four_gigabytes():
    """Offsets pass 32 bits: the last rows of 5.4 GB are those of a small call."""
    T, C = 1_320_000, 1024
    x = torch.empty(1, T, C, device=DEV)
    x.normal_()
    w = torch.randn(C, device=DEV)
    r, h = ops.residual_norm(x, x, (w, None, 1e-5), w, out_dtype=torch.bfloat16)
    for part in (slice(0, 700), slice(T - 700, T)):
        small = x[:, part].contiguous()
        r2, h2 = ops.residual_norm(small, small, (w, None, 1e-5), w, out_dtype=torch.bfloat16)
        assert torch.equal(r[:, part], r2)
        # Two kernels: each rounds to half a step, and each mean is off by a few 2^-24 of the row's largest value, which moves every
        # centred value of the row by as much, those near zero as well (as in Norm.check)
        r64 = r2.double()
        row = r64.abs().amax(-1, keepdim=True) / r64.std(-1, keepdim=True)
        close(h[:, part], h2.double(), torch.bfloat16, half_step(torch.bfloat16) * h2.double().abs() + 2 * 64 * F32 * row * w.double().abs(), "h")
    q, s = ops.quantize_tokens(h)
    q2, s2 = ops.quantize_tokens(h[:, -5:].contiguous())
    assert torch.equal(q[:, -5:], q2) and torch.equal(s[:, -5:], s2)
    del r, x, h
    wq = int8(40, C)
    ws = torch.ones(40, device=DEV)
    whole = q.repeat(1, 4, 1)                      # 5.4 GB of 8-bit tokens
    ss = s.repeat(1, 4)
    y = ops.int8_linear(whole, ss, wq, ws, None, torch.float32)
    assert torch.equal(y[:, -300:], ops.int8_linear(q[:, -300:].contiguous(), s[:, -300:].contiguous(), wq, ws, None, torch.float32))
