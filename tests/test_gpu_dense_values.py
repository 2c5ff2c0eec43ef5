"""Values that linear and qkv_norm_rope have to leave alone or carry through: infinities, NaN and -0 next to other columns, huge arguments."""
import math

import pytest
import torch

from speed3r_b200 import _lib, ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F16, FP32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(autouse=True)
def no_status():
    _lib.device_status()
    yield
    assert _lib.device_status() == 0


def same_bits(a, b):
    whole = torch.int32 if a.dtype == FP32 else torch.int16
    nan = torch.isnan(a)
    assert torch.equal(nan, torch.isnan(b))
    assert torch.equal(a.contiguous().view(whole)[~nan], b.contiguous().view(whole)[~nan])


# channels, axes, pairs: vectors of 4, 2 and 1 elements without a rotation, and with one of a part of the columns
STILL = [(64, 0, 0), (36, 0, 0), (50, 0, 0), (250, 0, 0), (80, 1, 20), (100, 1, 10), (66, 1, 15), (128, 2, 16), (254, 3, 5)]


@pytest.mark.parametrize("x", (BF16, F16, FP32))
@pytest.mark.parametrize("d, axes, pairs", STILL)
def test_columns_that_are_not_turned_are_their_own(d, axes, pairs, x):
    """Without a norm they leave as they came, forward and backward, whatever stands next to them; one special value per token."""
    g = torch.Generator(device=DEV).manual_seed(0)
    first, T = 2 * axes * pairs, 4 * (d - 2 * axes * pairs)
    rand = lambda *s: torch.randn(*s, device=DEV, generator=g).to(x)
    pos = torch.randint(0, 20, (1, T, axes), device=DEV, generator=g) if axes else None
    cos, sin = (rand(20, pairs), rand(20, pairs)) if axes else (None, None)
    clean = [rand(1, T, d) for _ in range(6)]                    # q, k, v and their gradients
    special = torch.tensor([math.inf, -math.inf, math.nan, -0.0], device=DEV).to(x).repeat(d - first)
    planted = [t.clone() for t in clean]
    for t in planted:
        t[0, torch.arange(T), first + torch.arange(T) // 4] = special
    results = []
    for q, k, v, dq, dk, dv in (clean, planted):
        qkv = torch.cat((q, k, v), -1).requires_grad_(True)
        out = ops.qkv_norm_rope(qkv, 1, 1, pos, cos, sin)
        back = torch.autograd.grad(out, qkv, [t[:, None] for t in (dq, dk, dv)])[0]
        results.append([o.detach()[:, 0] for o in out] + list(back.split(d, -1)))
    for i, (was, now) in enumerate(zip(*results)):
        still = slice(0 if i % 3 == 2 else first, d)             # v is never turned
        same_bits(now[..., still], planted[i][..., still])
        assert torch.equal(now[..., :first], was[..., :first])


@pytest.mark.parametrize("d, axes, pairs", STILL)
def test_parameters_of_columns_that_are_not_turned_are_their_own(d, axes, pairs):
    g = torch.Generator(device=DEV).manual_seed(1)
    rand = lambda *s: torch.randn(*s, device=DEV, generator=g)
    first, T = 2 * axes * pairs, 9
    qkv, w, b = rand(1, T, 3 * d).to(BF16), rand(d), rand(d)
    pos = torch.randint(0, 20, (1, T, axes), device=DEV, generator=g) if axes else None
    cos, sin = (rand(20, pairs), rand(20, pairs)) if axes else (None, None)
    call = lambda w, b: ops.qkv_norm_rope(qkv, 1, 1, pos, cos, sin, (w, b, 1e-5), (w, b, 1e-5))[:2]
    clean = call(w, b)
    for column in (first, first + 1, first + 3, (first + d) // 2, d - 1):
        for which in range(2):
            params = [w.clone(), b.clone()]
            params[which][column] = math.inf
            rest = torch.arange(d, device=DEV) != column
            for was, now in zip(clean, call(*params)):
                assert torch.isinf(now[..., column]).all() and torch.equal(now[..., rest], was[..., rest])


@pytest.mark.parametrize("scale", (False, True))
@pytest.mark.parametrize("act", ("gelu", "gelu_tanh", "silu"))
def test_slopes_as_far_out_as_bf16_reaches(act, scale):
    """z^2 is infinite in fp32 from 2^64 on: the activations are still z and 0 there, their slopes 1 and 0, exactly."""
    powers = [p for p in range(10, 124, 2)]
    M = 2 * len(powers)
    x = torch.zeros(M, 16, device=DEV, dtype=BF16)
    x[:, 0] = torch.tensor([sign * 2.0 ** p for p in powers for sign in (1, -1)], device=DEV)
    x.requires_grad_(True)
    w = torch.zeros(24, 16, device=DEV, dtype=BF16)
    w[:, 0] = 1
    s = torch.full((24,), 2.0, device=DEV, requires_grad=True) if scale else None
    y = ops.linear(x, w, torch.zeros(24, device=DEV), act=act, scale=s)
    factor = 2.0 if scale else 1.0
    assert torch.equal(y, factor * torch.relu(x[:, :1]).expand(M, 24))
    grads = torch.autograd.grad(y, [x] + ([s] if scale else []), torch.ones_like(y))
    assert torch.equal(grads[0][:, 0], 24.0 * factor * (x[:, 0] > 0)) and not grads[0][:, 1:].any()
    if scale:
        assert torch.allclose(grads[1].double(), torch.relu(x.double()[:, 0]).sum().expand(24), rtol=2.0 ** -20, atol=0)     # 57 additions of 2^-24


def test_a_sum_that_takes_seconds():
    """The longest that linear takes, made again in one part by the backward: no wait gives up on it (the status word is looked at)."""
    K = 2 ** 30 - 8
    x, w = torch.zeros(1, K, device=DEV, dtype=BF16), torch.zeros(1, K, device=DEV, dtype=BF16)
    x[0, 0], x[0, K // 2], x[0, -1] = 1.0, 2.0, -0.5
    w[0, 0], w[0, K // 2], w[0, -1] = 0.5, 0.25, 1.0
    b = torch.zeros(1, device=DEV, requires_grad=True)
    y = ops.linear(x, w, b, act="silu", out_dtype=FP32)
    db = torch.autograd.grad(y, b, torch.ones_like(y))[0]
    p = 1 / (1 + math.exp(-0.5))                                 # z = 0.5; the sigmoid within 2^-21
    assert abs(y.item() - 0.5 * p) <= 2.0 ** -20 and abs(db.item() - p * (1 + 0.5 * (1 - p))) <= 2.0 ** -19
