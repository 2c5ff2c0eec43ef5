"""The dense half of a block against plain 64-bit arithmetic: Linear layers with their epilogue, norms and rotation of q and k.

Tolerances: a rounding to a type is off by at most eps / 2 of the value (``close``).  In front of it:
* sums of K products: products of two 16-bit numbers are exact in fp32, every addition loses at most 2^-23 (the tensor cores cut off) of the
  magnitudes so far: K * 2^-23 * sum |x w|.
* activations: GELU's Phi within 7.5e-8 (the published bound) and ten roundings, the others' sigmoid within 2^-21: below 2^-20 |z| together; their
  slopes, which are at most 1.13 and change by at most 1 per unit, below 2^-19.
* dz is rounded to the operands' type in front of its two products: half a step of it."""
import itertools
import math

import pytest
import torch

from speed3r_b200 import _lib, ops
from test_gpu_block_ops import F32, close, half_step

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F16, FP32 = torch.bfloat16, torch.float16, torch.float32
ACTS = (None, "gelu", "gelu_tanh", "silu")


@pytest.fixture(autouse=True)
def no_status():
    _lib.device_status()
    yield
    assert _lib.device_status() == 0


def act64(z, act):
    """(act(z), slope)"""
    if act is None:
        return z, torch.ones_like(z)
    if act == "gelu":
        below = 0.5 * torch.special.erfc(-z / math.sqrt(2))
        return z * below, below + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    w, dw = (z, 1) if act == "silu" else (2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3), 2 * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * z * z))
    p = torch.sigmoid(w)
    return z * p, p + z * p * (1 - p) * dw


class Linear:
    def __init__(self, M, N, K, x=BF16, act=None, bias=None, scale=None, residual=None, out=None, lead=None, seed=0):
        g = torch.Generator(device=DEV).manual_seed(seed)
        rand = lambda *s: torch.randn(*s, device=DEV, generator=g)
        lead = (M,) if lead is None else lead
        self.x, self.w = rand(*lead, K).to(x), (rand(N, K) / math.sqrt(K)).to(x)
        self.bias = None if bias is None else (0.3 * rand(N)).to(bias)
        self.scale = None if scale is None else (0.5 * rand(N)).to(scale)
        self.residual = None if residual is None else (2 * rand(*lead, N)).to(residual)
        self.act, self.out = act, out
        self.type = out or (x if residual is None else residual)
        self.dy = rand(*lead, N).to(self.type)

    def leaves(self):
        return {n: t for n, t in (("x", self.x), ("w", self.w), ("bias", self.bias), ("scale", self.scale), ("residual", self.residual)) if t is not None}

    def call(self):
        return ops.linear(self.x, self.w, self.bias, self.act, self.residual, self.scale, self.out)

    def check(self, y, grads=None):
        N, K = self.w.shape
        x, w, t = self.x.detach().double().reshape(-1, K), self.w.detach().double(), self.x.dtype
        M = x.shape[0]
        b, s = (torch.full((N,), float(o), dtype=torch.float64, device=DEV) if v is None else v.detach().double() for v, o in ((self.bias, 0), (self.scale, 1)))
        z = x @ w.T + b
        z_far = 2 * F32 * (K + 2) * (x.abs() @ w.abs().T + b.abs())
        u, slope = act64(z, self.act)
        u_far = 1.13 * z_far + (z.abs() * 2.0 ** -20 if self.act else 0)
        r = self.residual.detach().double().reshape(-1, N) if self.residual is not None else torch.zeros_like(z)
        close(y.reshape(-1, N), u * s + r, self.type, u_far * s.abs() + 4 * F32 * ((u * s).abs() + r.abs()), "y")
        assert y.shape == self.x.shape[:-1] + (N,)
        if grads is None:
            return
        dy = self.dy.double().reshape(-1, N)
        du = dy * s
        dz = du * slope
        dz_far = du.abs() * (z_far + 2.0 ** -19 if self.act else 4 * F32) + 4 * F32 * dz.abs()
        kept = dz_far + half_step(t) * (dz.abs() + torch.finfo(t).tiny)
        if "x" in grads:
            close(grads["x"].reshape(-1, K), dz @ w, t, kept @ w.abs() + 2 * F32 * (N + 2) * ((dz.abs() + kept) @ w.abs()), "dx")
        if "w" in grads:
            close(grads["w"], dz.T @ x, t, kept.T @ x.abs() + 2 * F32 * (M + 2) * ((dz.abs() + kept).T @ x.abs()), "dw")
        if "bias" in grads:
            close(grads["bias"], dz.sum(0), self.bias.dtype, dz_far.sum(0) + M * F32 * dz.abs().sum(0), "dbias")
        if "scale" in grads:
            close(grads["scale"], (dy * u).sum(0), self.scale.dtype, (dy.abs() * u_far).sum(0) + (M + 4) * F32 * (dy * u).abs().sum(0), "dscale")
        if "residual" in grads:
            assert torch.equal(grads["residual"], self.dy.to(self.residual.dtype))

    def train(self, *frozen):
        leaves = {n: t.requires_grad_(True) for n, t in self.leaves().items() if n not in frozen}
        y = self.call()
        grads = dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), self.dy)))
        for n, t in leaves.items():
            assert grads[n].dtype == t.dtype and grads[n].shape == t.shape, n
        self.check(y, grads)
        return y, grads


# one element; odd everything; the few-token kernel at its edges; single CTAs and pairs of either width; ragged tiles; several tiles per CTA
SIZES = [(1, 1, 1), (1, 4096, 1024), (2, 33, 8), (3, 5, 7), (8, 130, 520), (9, 64, 64), (31, 40, 200), (64, 1024, 512), (129, 257, 65), (128, 128, 64),
         (300, 500, 1023), (257, 24, 2048), (1041, 1543, 517), (700, 2048, 96), (2600, 1792, 128)]


@pytest.mark.parametrize("size, act", [(s, ACTS[i % 4]) for i, s in enumerate(SIZES)] + [((65, 96, 72), a) for a in ACTS])
def test_linear_forward(size, act):
    i = SIZES.index(size) if size in SIZES else 3
    x = (BF16, F16)[i % 2]
    Linear(*size, x=x, act=act).check(Linear(*size, x=x, act=act).call())
    c = Linear(*size, x=x, act=act, bias=FP32, scale=FP32, residual=FP32, seed=1)
    c.check(c.call())
    c = Linear(*size, x=x, act=act, bias=x, residual=(F16, BF16)[i % 2], scale=(x, BF16)[i // 2 % 2], out=(None, FP32, BF16)[i % 3], seed=2)
    c.check(c.call())


@pytest.mark.parametrize("size, act", [(s, ACTS[(i + 1) % 4]) for i, s in enumerate(SIZES)] + [((65, 96, 72), a) for a in ACTS])
def test_linear_gradients(size, act):
    i = SIZES.index(size) if size in SIZES else 3
    x = (F16, BF16)[i % 2]
    Linear(*size, x=x, act=act, bias=FP32).train()
    Linear(*size, x=x, act=act, bias=x, scale=FP32, residual=FP32, seed=1).train()
    Linear(*size, x=x, act=act, scale=x, out=FP32, seed=2).train()
    Linear(*size, x=x, seed=3).train()


def test_linear_gradients_of_some():
    """What is frozen gets no gradient, and the rest the same."""
    names = ("x", "w", "bias", "scale", "residual")
    whole = Linear(70, 100, 40, act="gelu", bias=FP32, scale=FP32, residual=FP32).train()[1]
    for n in range(1, 5):
        for frozen in itertools.combinations(names, n):
            some = Linear(70, 100, 40, act="gelu", bias=FP32, scale=FP32, residual=FP32).train(*frozen)[1]
            assert set(some) == set(names) - set(frozen)
            for k, t in some.items():
                assert torch.equal(t, whole[k]), (frozen, k)
    for frozen in (("x",), ("w",), ("x", "w"), ("scale",), ("x", "w", "bias")):
        Linear(70, 100, 40, bias=FP32, scale=FP32).train(*frozen)


def test_linear_gradient_against_differences():
    """(L(w + h v) - L(w - h v)) / 2h of the forward itself, in directions of every leaf; the result in fp32."""
    g = torch.Generator(device=DEV).manual_seed(5)
    for act in ACTS:
        c = Linear(40, 24, 32, act=act, bias=FP32, scale=FP32, residual=FP32, out=FP32)
        _, grads = Linear(40, 24, 32, act=act, bias=FP32, scale=FP32, residual=FP32, out=FP32).train()
        for name in ("bias", "scale", "residual"):
            leaf = c.leaves()[name]
            v, h = torch.randn(leaf.shape, device=DEV, generator=g), 2.0 ** -6
            ends = []
            for sign in (1, -1):
                kept = leaf.clone()
                leaf.add_(v, alpha=sign * h)
                ends.append((c.call().double() * c.dy.double()).sum())
                leaf.copy_(kept)
            got, want = (ends[0] - ends[1]) / (2 * h), (grads[name].double() * v.double()).sum()
            # third derivatives of the activations are below 2: h^2 / 6 * 2 * sum |dy s v^3|; fp32 values of the forward over 2 h
            total = (c.dy.double().abs().sum(0) * c.scale.double().abs() * v.double().abs().amax() ** 3).sum()
            y = c.call().double()
            assert (got - want).abs() <= h * h / 3 * total + 64 * F32 * (y.abs() * c.dy.double().abs()).sum() / h, (act, name)


def test_linear_rows_that_lie_elsewhere():
    """Slices, offsets, transposed and broadcast operands, leading dimensions: the result of contiguous ones, bit for bit."""
    c = Linear(90, 72, 136, act="silu", bias=FP32, residual=BF16, scale=BF16)
    want = c.call()
    c.check(want)
    wide = torch.full((90, 200), math.nan, device=DEV, dtype=BF16)
    for first in (0, 8, 3):                                      # at multiples of 16 bytes, and not
        x = wide[:, first:first + 136]
        x.copy_(c.x)
        assert torch.equal(ops.linear(x, c.w, c.bias, c.act, c.residual, c.scale), want)
        w = wide[:72, first:first + 136]
        w.copy_(c.w)
        assert torch.equal(ops.linear(c.x, w, c.bias, c.act, c.residual, c.scale), want)
    odd = torch.full((90 * 137 + 1,), math.nan, device=DEV, dtype=BF16)[1:].view(90, 137)[:, :136]
    odd.copy_(c.x)
    assert torch.equal(ops.linear(odd, c.w, c.bias, c.act, c.residual, c.scale), want)
    assert torch.equal(ops.linear(c.x.T.contiguous().T, c.w.T.contiguous().T, c.bias, c.act, c.residual.T.contiguous().T, c.scale), want)
    assert torch.equal(ops.linear(c.x.view(2, 3, 15, 136), c.w, c.bias, c.act, c.residual.view(2, 3, 15, 72), c.scale), want.view(2, 3, 15, 72))
    row = ops.linear(c.x[:1], c.w, c.bias, c.act)
    same = ops.linear(c.x[0].expand(20, 136), c.w, c.bias, c.act)
    close(same, row.double().expand(20, 72), BF16, half_step(BF16) * row.double().abs() + 2.0 ** -12)
    assert torch.equal(ops.linear(c.x[0], c.w, c.bias, c.act), row[0])
    stride = torch.randn(72, 2, device=DEV)
    assert torch.equal(ops.linear(c.x, c.w, stride[:, 0]), ops.linear(c.x, c.w, stride[:, 0].contiguous()))
    x = c.x.T.contiguous().T.requires_grad_(True)
    dy = torch.randn(72, 90, device=DEV).to(BF16).T
    y = ops.linear(x, c.w, act="gelu")
    got = torch.autograd.grad(y, x, dy)[0]
    z = Linear(90, 72, 136, act="gelu")
    z.dy = dy.contiguous()
    assert torch.equal(got, torch.autograd.grad(ops.linear(z.x.requires_grad_(True), z.w, act="gelu"), z.x, z.dy)[0])


def test_linear_without_rows():
    c = Linear(0, 40, 24, act="gelu", bias=FP32, scale=FP32, residual=FP32)
    y, grads = c.train()
    assert y.shape == (0, 40) and all(not g.any() for g in grads.values())
    assert ops.linear(torch.empty(3, 0, 24, device=DEV, dtype=BF16), c.w).shape == (3, 0, 40)


@pytest.mark.parametrize("M", (5, 200))
def test_linear_infinities_and_nan_stay_in_their_rows_and_columns(M):
    for act in ACTS:
        c = Linear(M, 70, 64, act=act, bias=FP32, residual=FP32, scale=FP32)
        clean = c.call()
        c.x[1, 3], c.x[2, 5] = math.nan, math.inf
        c.bias[7], c.bias[8] = math.inf, -math.inf
        y = c.call()
        z = (c.x.double() @ c.w.double().T + c.bias.double()).float()
        # infinity times nothing is NaN, as in the formulas
        if act == "gelu":
            u = 0.5 * z * (1 + torch.erf(z / math.sqrt(2)))
        elif act == "gelu_tanh":
            u = 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
        else:
            u = z * torch.sigmoid(z) if act else z
        want = c.residual + u * c.scale
        assert torch.equal(torch.isnan(y), torch.isnan(want)), act
        assert torch.equal(y[torch.isinf(want)], want[torch.isinf(want)]), act
        rows = torch.ones(M, dtype=torch.bool, device=DEV)
        rows[1:3] = False
        columns = torch.ones(70, dtype=torch.bool, device=DEV)
        columns[7:9] = False
        assert torch.equal(y[rows][:, columns], clean[rows][:, columns])


def test_linear_sums_ignore_rows_that_are_not_there():
    """A weight that is infinite makes NaN of the zeros behind the last row; they are not counted."""
    c = Linear(33, 64, 64, act="silu", bias=FP32, scale=FP32)
    _, clean = Linear(33, 64, 64, act="silu", bias=FP32, scale=FP32).train()
    c.w[5, 0] = math.inf
    leaves = [c.bias.requires_grad_(True), c.scale.requires_grad_(True)]
    db, ds = torch.autograd.grad(c.call(), leaves, c.dy)
    assert not torch.isfinite(ds[5]) and torch.equal(torch.cat((db[:5], db[6:])), torch.cat((clean["bias"][:5], clean["bias"][6:])))
    assert torch.equal(torch.cat((ds[:5], ds[6:])), torch.cat((clean["scale"][:5], clean["scale"][6:])))


def test_linear_beyond_32_bits():
    """Rows whose elements' numbers pass 2^31, in x, in the result and in the gradients."""
    M, N, K = 530_000, 4104, 16
    g = torch.Generator(device=DEV).manual_seed(0)
    x, w = torch.randn(M, K, device=DEV, generator=g).to(BF16), torch.randn(N, K, device=DEV, generator=g).to(BF16)
    assert M * N > 2 ** 31
    y = ops.linear(x, w, act="gelu")
    for rows in (slice(0, 3), slice(M - 300, M)):
        assert torch.equal(y[rows], ops.linear(x[rows].repeat(1 + 16 // x[rows].shape[0], 1), w, act="gelu")[:x[rows].shape[0]])
    dx = torch.autograd.grad(ops.linear(x.requires_grad_(True), w, act="gelu"), x, y)[0]
    # few rows take their sums in parts: N products in another order, each addition off by at most 2^-23 of the magnitudes, and two roundings
    tail = x.detach()[-300:].requires_grad_(True)
    want = torch.autograd.grad(ops.linear(tail, w, act="gelu"), tail, y[-300:])[0].double()
    size = 1.13 * y[-300:].double().abs() @ w.double().abs()
    assert ((dx[-300:].double() - want).abs() <= 4 * F32 * (N + 2) * size + 2 * half_step(BF16) * want.abs()).all()
    del y, dx, x
    x = torch.zeros(N, M, device=DEV, dtype=BF16)                                          # as an operand
    x[-1], x[-2, ::2] = 1.0, 1.0
    one = torch.ones(1, M, device=DEV, dtype=BF16)
    assert ops.linear(x, one, out_dtype=FP32)[-3:, 0].tolist() == [0.0, M / 2, float(M)]


def test_linear_repeats_its_bits():
    c = Linear(700, 520, 264, act="gelu", bias=FP32, scale=FP32, residual=FP32)
    y, g = c.train()
    for _ in range(3):
        y2, g2 = c.train()
        assert torch.equal(y, y2) and all(torch.equal(g[k], g2[k]) for k in g)


def test_linear_on_a_stream_and_in_a_graph():
    c = Linear(300, 256, 200, act="gelu", bias=FP32, scale=FP32, residual=FP32)
    leaves = [t.requires_grad_(True) for t in c.leaves().values()]
    call = lambda: torch.autograd.grad(c.call(), leaves, c.dy)
    want = [c.call().detach()] + list(call())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [c.call().detach()] + list(call())
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs, kept = [], []
    for _ in range(2):                                            # two of them, replayed in turn
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            kept.append([c.call().detach()] + list(call()))
        graphs.append(graph)
    with torch.no_grad():
        c.x.mul_(0.5)
        c.dy.mul_(2.0)
    want = [c.call().detach()] + list(call())
    for graph in graphs + graphs:
        graph.replay()
    for outs in kept:
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


# ---- q, k and v ------------------------------------------------------------------------------------------------------------
class Qkv:
    def __init__(self, B, T, H, Hk, d, x=BF16, w=FP32, kind="layer", norms="qk", affine="wb", axes=2, pairs=None, rows=40, table=FP32, seed=0):
        g = torch.Generator(device=DEV).manual_seed(seed)
        rand = lambda *s: torch.randn(*s, device=DEV, generator=g)
        self.H, self.Hk, self.d, self.kind = H, Hk, d, kind
        self.qkv = (rand(B, T, (H + 2 * Hk) * d) + 0.3).to(x)
        one = lambda n: ((1 + 0.3 * rand(d)).to(w) if "w" in affine else None, (0.3 * rand(d)).to(w) if "b" in affine else None, 1e-5) if n in norms else None
        self.norms = [one("q"), one("k")]
        self.pos = self.cos = self.sin = None
        if axes:
            self.W = d // (2 * axes) if pairs is None else pairs
            self.pos = torch.randint(0, rows, (B, T, axes), device=DEV, generator=g)
            angle = 7 * rand(rows, self.W)
            self.cos, self.sin = angle.cos().to(table), angle.sin().to(table)
        self.grads = [rand(B, h, T, d).to(x) for h in (H, Hk, Hk)]

    def leaves(self):
        named = {"qkv": self.qkv}
        for n, norm in zip("qk", self.norms):
            if norm:
                named.update({n + "w": norm[0], n + "b": norm[1]})
        return {n: t for n, t in named.items() if t is not None}

    def call(self):
        return ops.qkv_norm_rope(self.qkv, self.H, self.Hk, self.pos, self.cos, self.sin, *self.norms, self.kind)

    def turn(self, x, back=False, sizes=False):
        """x [B, T, h, d] rotated; ``sizes``: the magnitudes that go into it."""
        if self.pos is None:
            return x
        out = x.clone()
        for a in range(self.pos.shape[-1]):
            c, s = (t.double()[self.pos[..., a]][:, :, None] for t in (self.cos, self.sin))
            i = 2 * self.W * a
            x1, x2 = x[..., i:i + self.W], x[..., i + self.W:i + 2 * self.W]
            if sizes:
                c, s = c.abs(), s.abs()
                out[..., i:i + self.W], out[..., i + self.W:i + 2 * self.W] = x1 * c + x2 * s, x2 * c + x1 * s
            else:
                s = -s if back else s
                out[..., i:i + self.W], out[..., i + self.W:i + 2 * self.W] = x1 * c - x2 * s, x2 * c + x1 * s
        return out

    def check(self, out, grads=None):
        B, T, _ = self.qkv.shape
        t, tiny = self.qkv.dtype, 64 * F32
        parts = self.qkv.detach().double().view(B, T, self.H + 2 * self.Hk, self.d).split((self.H, self.Hk, self.Hk), 2)
        assert torch.equal(out[2], self.qkv.detach().view(B, T, self.H + 2 * self.Hk, self.d)[:, :, -self.Hk:].transpose(1, 2)) and all(o.is_contiguous() for o in out)
        far_qkv, d_qkv = [], []
        for i, (x, norm, n) in enumerate(zip(parts, self.norms + [None], "qkv")):
            heads = x.shape[2]
            w = norm[0].detach().double() if norm and norm[0] is not None else torch.ones(self.d, dtype=torch.float64, device=DEV)
            b = norm[1].detach().double() if norm and norm[1] is not None else torch.zeros(self.d, dtype=torch.float64, device=DEV)
            unit, inv, row = x, None, 0
            if norm:
                mean = x.mean(-1, keepdim=True) if self.kind == "layer" else 0
                inv = 1 / torch.sqrt(((x - mean) ** 2).mean(-1, keepdim=True) + norm[2])
                unit, row = (x - mean) * inv, x.abs().amax(-1, keepdim=True) * inv
            h = unit * w + b
            if n != "v":
                far = tiny * ((row + unit.abs()) * w.abs() + b.abs()) if norm else 0 * x
                close(out[i], self.turn(h).transpose(1, 2), t, (self.turn(far, sizes=True) + 4 * F32 * self.turn(h.abs(), sizes=True)).transpose(1, 2), n)
            if grads is None:
                continue
            dy = self.grads[i].double().transpose(1, 2)
            dh, dh_far = (dy, 0 * dy) if n == "v" else (self.turn(dy, back=True), 4 * F32 * self.turn(dy.abs(), sizes=True))
            if not norm:
                d_qkv.append(dh), far_qkv.append(dh_far)
                continue
            sums = lambda v: v.sum((0, 1, 2))
            count = B * T * heads
            if n + "w" in grads:
                close(grads[n + "w"], sums(dh * unit), norm[0].dtype,
                      sums(dh.abs() * tiny * (row + unit.abs()) + dh_far * unit.abs()) + (tiny + count * F32) * sums((dh * unit).abs()), "d" + n + "w")
            if n + "b" in grads:
                close(grads[n + "b"], sums(dh), norm[1].dtype, sums(dh_far) + (tiny + count * F32) * sums(dh.abs()), "d" + n + "b")
            e = dh * w
            flat = e.mean(-1, keepdim=True) if self.kind == "layer" else 0
            dx = inv * (e - flat - unit * (e * unit).mean(-1, keepdim=True))
            big = inv * (e.abs() + dh_far * w.abs()).amax(-1, keepdim=True) * (1 + unit.abs()) * (1 + row)
            d_qkv.append(dx), far_qkv.append(tiny * (big + dx.abs()))
        if grads is not None:
            close(grads["qkv"], torch.cat(d_qkv, 2).flatten(2), t, torch.cat(far_qkv, 2).flatten(2), "dqkv")

    def train(self):
        leaves = {n: t.requires_grad_(True) for n, t in self.leaves().items()}
        out = self.call()
        grads = dict(zip(leaves, torch.autograd.grad(out, list(leaves.values()), self.grads)))
        self.check(out, grads)
        return out, grads


# vectors of 8 by 2, 4, 8 and 16 threads with idle ones among them, of 4, and single elements; one token; several chunks of heads and rounds of tokens
HEADS = [(1, 1, 16, 16, 64, {}), (2, 33, 3, 1, 64, {}), (1, 70, 4, 2, 16, dict(axes=1)), (3, 41, 2, 2, 96, dict(axes=2)), (1, 50, 6, 3, 128, dict(axes=1)),
         (1, 19, 2, 1, 256, dict(axes=2)), (2, 37, 3, 3, 80, dict(axes=1, pairs=20)), (1, 45, 2, 1, 72, dict(axes=3)), (1, 45, 4, 1, 48, dict(axes=2)),
         (2, 29, 2, 2, 2, dict(axes=1)), (1, 61, 3, 1, 26, dict(axes=1)), (1, 23, 2, 1, 254, dict(axes=3, pairs=5)), (1, 40, 5, 5, 64, dict(axes=0)),
         (2, 600, 16, 16, 64, {}), (1, 40, 3, 1, 250, dict(axes=0)), (1, 40, 3, 1, 200, dict(axes=2, pairs=12)), (1, 35, 2, 2, 64, dict(axes=4, pairs=8))]


@pytest.mark.parametrize("case", range(len(HEADS)))
@pytest.mark.parametrize("x", (BF16, F16, FP32))
def test_qkv_forward_and_gradients(case, x):
    *sizes, more = HEADS[case]
    turn = case + (BF16, F16, FP32).index(x)
    kind, w = ("layer", "rms")[turn % 2], (FP32, x)[turn // 2 % 2]
    c = Qkv(*sizes, x=x, w=w, kind=kind, affine=("wb", "w", "wb", "")[turn % 4], table=(FP32, x)[turn % 2], **more)
    with torch.no_grad():
        c.check(c.call())
    c.train()
    Qkv(*sizes, x=x, w=w, kind=kind, norms=("", "q", "k")[turn % 3], table=(x, FP32)[turn % 2], seed=1, **more).train()


def test_qkv_gradient_against_differences():
    """(L(p + h v) - L(p - h v)) / 2h of the forward itself, fp32."""
    g = torch.Generator(device=DEV).manual_seed(5)
    for kind in ("layer", "rms"):
        c = Qkv(1, 24, 2, 1, 32, x=FP32, kind=kind)
        _, grads = Qkv(1, 24, 2, 1, 32, x=FP32, kind=kind).train()
        for name, leaf in c.leaves().items():
            v, h = torch.randn(leaf.shape, device=DEV, generator=g), 2.0 ** -7
            value = lambda: sum((o.double() * d.double()).sum() for o, d in zip(c.call(), c.grads))
            kept, ends = leaf.clone(), []
            for sign in (1, -1):
                leaf.copy_(kept + sign * h * v)
                ends.append(value())
                leaf.copy_(kept)
            got, want = (ends[0] - ends[1]) / (2 * h), (grads[name].double() * v.double()).sum()
            # fp32 of the forward over 2 h; the norm's third derivative along v: at most 16 |v / sigma|^3 of a value for |v| below 4 sigma
            size = sum((o.double().abs() * d.double().abs()).sum() for o, d in zip(c.call(), c.grads))
            slack = 64 * F32 * size / h + (h * h * 16 * 8 * size if name == "qkv" else 64 * F32 * size)
            assert (got - want).abs() <= slack, (kind, name, float(got), float(want))


def test_qkv_that_lies_elsewhere():
    """Slices of a wider matrix, offsets that are multiples of nothing, positions of one sample for all, strided gradients and tables."""
    c = Qkv(3, 21, 4, 2, 64)
    want, grads = c.train()
    C = c.qkv.shape[-1]
    c.qkv = c.qkv.detach()
    wide = torch.full((3, 30, C + 40), math.nan, device=DEV, dtype=BF16)
    for first in (0, 8, 5):
        view = wide[:, 4:25, first:first + C]
        view.copy_(c.qkv)
        view.requires_grad_(False)
        got = ops.qkv_norm_rope(view, 4, 2, c.pos, c.cos, c.sin, *c.norms)
        c.check(got)
        # at multiples of 16 bytes in the same vectors, whose sums have the same order; elsewhere in another, within the bounds of check()
        assert first == 5 or all(torch.equal(a, b) for a, b in zip(got, want))
    turned = c.qkv.permute(2, 1, 0).contiguous().permute(2, 1, 0)
    assert all(torch.equal(a, b) for a, b in zip(ops.qkv_norm_rope(turned, 4, 2, c.pos, c.cos, c.sin, *c.norms), want))
    twice = torch.cat((c.cos, c.cos), 1), torch.cat((c.sin, c.sin), 1)          # as RoPE2D keeps them
    assert all(torch.equal(a, b) for a, b in zip(ops.qkv_norm_rope(c.qkv, 4, 2, c.pos, twice[0][:, :c.W], twice[1][:, :c.W], *c.norms), want))
    assert all(torch.equal(a, b) for a, b in zip(ops.qkv_norm_rope(c.qkv, 4, 2, c.pos.int(), c.cos, c.sin, *c.norms), want))
    one = c.pos[:1]
    of = lambda p: ops.qkv_norm_rope(c.qkv, 4, 2, p, c.cos, c.sin, *c.norms)
    for p in (one, one[0], one.permute(2, 0, 1).contiguous().permute(1, 2, 0)):
        assert all(torch.equal(a, b) for a, b in zip(of(p), of(one.repeat(3, 1, 1))))
    x = c.qkv.clone().requires_grad_(True)
    out = ops.qkv_norm_rope(x, 4, 2, c.pos, c.cos, c.sin, *c.norms)
    strided = [g.transpose(1, 2).contiguous().transpose(1, 2) for g in c.grads]     # [B, T, H, d] in memory, as attention leaves them
    assert torch.equal(torch.autograd.grad(out, x, strided)[0], grads["qkv"])
    out = ops.qkv_norm_rope(x, 4, 2, c.pos, c.cos, c.sin, *c.norms)
    flat = [g.transpose(2, 3).contiguous().transpose(2, 3) for g in c.grads]
    assert torch.equal(torch.autograd.grad(out, x, flat)[0], grads["qkv"])


def test_qkv_gradients_that_are_missing():
    c = Qkv(2, 17, 4, 2, 64)
    for some in ((0,), (1,), (2,), (0, 2)):
        x = c.qkv.detach().clone().requires_grad_(True)
        out = ops.qkv_norm_rope(x, 4, 2, c.pos, c.cos, c.sin, *c.norms)
        got = torch.autograd.grad([out[i] for i in some], x, [c.grads[i] for i in some])[0]
        out = ops.qkv_norm_rope(x, 4, 2, c.pos, c.cos, c.sin, *c.norms)
        assert torch.equal(got, torch.autograd.grad(out, x, [g if i in some else torch.zeros_like(g) for i, g in enumerate(c.grads)])[0])
    frozen = Qkv(2, 17, 4, 2, 64)
    frozen.norms[0][0].requires_grad_(True)
    got = torch.autograd.grad(frozen.call(), frozen.norms[0][0], frozen.grads)[0]
    assert torch.equal(got, Qkv(2, 17, 4, 2, 64).train()[1]["qw"])


def test_qkv_without_tokens():
    c = Qkv(2, 0, 4, 2, 64)
    out, grads = c.train()
    assert out[0].shape == (2, 4, 0, 64) and all(not g.any() for g in grads.values())


def test_qkv_position_outside_of_the_tables_is_flagged():
    c = Qkv(1, 20, 2, 2, 64, rows=30)
    c.pos[0, 3, 0], c.pos[0, 4, 1] = 30, -1
    got = c.call()
    assert _lib.device_status() == 2
    c.pos[0, 3, 0], c.pos[0, 4, 1] = 29, 0
    assert all(torch.equal(a, b) for a, b in zip(got, c.call()))


def test_qkv_nan_stays_in_its_head():
    c = Qkv(1, 12, 3, 1, 64)
    clean = c.call()
    c.qkv[0, 5, 64 + 7] = math.nan
    c.qkv[0, 6, 2 * 64] = math.inf
    got = c.call()
    assert torch.isnan(got[0][0, 1, 5]).all() and not torch.isfinite(got[0][0, 2, 6]).any()
    got[0][0, 1, 5], got[0][0, 2, 6] = clean[0][0, 1, 5], clean[0][0, 2, 6]
    assert all(torch.equal(a, b) for a, b in zip(got, clean))


def test_qkv_beyond_32_bits():
    B, T, H, Hk, d = 1, 850_000, 12, 4, 128
    g = torch.Generator(device=DEV).manual_seed(0)
    x = torch.empty(B, T, (H + 2 * Hk) * d, device=DEV, dtype=BF16)
    assert x.numel() > 2 ** 31
    x[:, :100].normal_(generator=g)
    x[:, -100:].normal_(generator=g)
    c = Qkv(1, 200, H, Hk, d, axes=1)
    pos = torch.zeros(B, T, 1, dtype=torch.int64, device=DEV)
    pos[:, :100], pos[:, -100:] = c.pos[:, :100], c.pos[:, 100:]
    ends = torch.cat((x[:, :100], x[:, -100:]), 1)
    leaf = x.requires_grad_(True)
    out = ops.qkv_norm_rope(leaf, H, Hk, pos, c.cos, c.sin, *c.norms)
    small = ends.requires_grad_(True)
    want = ops.qkv_norm_rope(small, H, Hk, c.pos, c.cos, c.sin, *c.norms)
    for a, b in zip(out, want):
        assert torch.equal(torch.cat((a[:, :, :100], a[:, :, -100:]), 2), b)
    grads = [torch.zeros_like(o) for o in out]
    for big, g in zip(grads, c.grads):
        big[:, :, :100], big[:, :, -100:] = g[:, :, :100], g[:, :, 100:]
    got = torch.autograd.grad(out, leaf, grads)[0]
    assert torch.equal(torch.cat((got[:, :100], got[:, -100:]), 1), torch.autograd.grad(want, small, c.grads)[0])


def test_qkv_on_a_stream_and_in_a_graph():
    c = Qkv(2, 300, 4, 4, 64)
    leaves = [t.requires_grad_(True) for t in c.leaves().values()]
    call = lambda: [o.detach() for o in c.call()] + list(torch.autograd.grad(c.call(), leaves, c.grads))
    want = call()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = call()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs, kept = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            kept.append(call())
        graphs.append(graph)
    with torch.no_grad():
        c.qkv.mul_(0.5).add_(0.1)
    want = call()
    for graph in graphs + graphs:
        graph.replay()
    for outs in kept:
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


# ---- as they are used together -------------------------------------------------------------------------------------------------
def test_a_block_of_them():
    """qkv, norms and rotation, attention, projection with LayerScale and residual, norm, MLP: forward and gradients against 64 bits.  Every step
    rounds to bf16, seven of them one behind the other, so that values of about 1 are off by a few half steps of it."""
    B, T, C, H = 2, 50, 128, 2
    g = torch.Generator(device=DEV).manual_seed(3)
    rand = lambda *s: torch.randn(*s, device=DEV, generator=g)
    shapes = dict(qkv=(3 * C, C), proj=(C, C), up=(4 * C, C), down=(C, 4 * C))
    w = {n: (rand(*s) / math.sqrt(s[1])).to(BF16).requires_grad_(True) for n, s in shapes.items()}
    b = {n: (0.1 * rand(s[0])).requires_grad_(True) for n, s in shapes.items()}
    one = lambda n: [(1 + 0.1 * rand(n)).requires_grad_(True), (0.1 * rand(n)).requires_grad_(True)]
    n1, n2, qn, kn = one(C), one(C), one(64), one(64)
    ls = [(0.5 * rand(C)).requires_grad_(True) for _ in range(2)]
    x0 = rand(B, T, C).requires_grad_(True)
    pos = torch.randint(0, 30, (B, T, 2), device=DEV, generator=g)
    angle = rand(30, 16) * 3
    dy = rand(B, T, C)

    def own():
        _, h = ops.residual_norm(x0, None, (*n1, 1e-5), out_dtype=BF16)
        q, k, v = ops.qkv_norm_rope(ops.linear(h, w["qkv"], b["qkv"]), H, None, pos, angle.cos(), angle.sin(), (*qn, 1e-5), (*kn, 1e-5))
        a = torch.nn.functional.scaled_dot_product_attention(q, k, v).transpose(1, 2).reshape(B, T, C)
        x = ops.linear(a, w["proj"], b["proj"], residual=x0, scale=ls[0])
        _, h = ops.residual_norm(x, None, (*n2, 1e-5), out_dtype=BF16)
        return ops.linear(ops.linear(h, w["up"], b["up"], "gelu"), w["down"], b["down"], residual=x, scale=ls[1])

    def plain(of):
        norm = lambda x, p: torch.nn.functional.layer_norm(x, x.shape[-1:], of(p[0]), of(p[1]), 1e-5)
        lin = lambda x, n: x @ of(w[n]).T + of(b[n])

        def turn(x):
            out = []
            for a in range(2):
                c, s = (t[pos[..., a]][:, :, None] for t in (of(angle).cos(), of(angle).sin()))
                x1, x2 = x[..., 32 * a:32 * a + 16], x[..., 32 * a + 16:32 * a + 32]
                out += [x1 * c - x2 * s, x2 * c + x1 * s]
            return torch.cat(out, -1)
        x = of(x0)
        q, k, v = lin(norm(x, n1), "qkv").view(B, T, 3, H, 64).unbind(2)
        q, k, v = (t.transpose(1, 2) for t in (turn(norm(q, qn)), turn(norm(k, kn)), v))
        a = (torch.softmax(q @ k.transpose(2, 3) / 8, -1) @ v).transpose(1, 2).reshape(B, T, C)
        x = x + lin(a, "proj") * of(ls[0])
        h = lin(norm(x, n2), "up")
        return x + lin(h * 0.5 * torch.special.erfc(-h / math.sqrt(2)), "down") * of(ls[1])

    leaves = [x0, *w.values(), *b.values(), *n1, *n2, *qn, *kn, *ls]
    y = own()
    want = plain(lambda t: t.double())
    got = torch.autograd.grad(y, leaves, dy)
    ref = torch.autograd.grad(want, leaves, dy.double())
    step = half_step(BF16)
    for a, r in zip((y, *got), (want, *ref)):
        size = r.double().pow(2).mean().sqrt()
        off = (a.double() - r.double()).pow(2).mean().sqrt()
        assert off <= 8 * step * size, (a.shape, float(off / size))
