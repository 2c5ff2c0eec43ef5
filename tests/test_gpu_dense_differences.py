"""Gradients of linear's 16-bit operands against differences of its own forward.

Operands lie on a grid that leaves bits for the step, so that both ends are exact in their type; the step has the gradient's signs, and the difference
of the ends is then the sum of its magnitudes."""
import pytest
import torch

from speed3r_b200 import _lib
from test_gpu_block_ops import F32, half_step
from test_gpu_dense_ops import ACTS, BF16, F16, FP32, Linear, act64

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def no_status():
    _lib.device_status()
    yield
    assert _lib.device_status() == 0


# whole tiles of one CTA and of a pair, and rows and columns that are multiples of nothing
@pytest.mark.parametrize("size", [(40, 24, 32), (37, 41, 35), (300, 136, 72), (5, 30, 200)])
@pytest.mark.parametrize("name", ("x", "w"))
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("t", (BF16, F16))
def test_operands_against_differences(size, name, act, t):
    c = Linear(*size, x=t, act=act, bias=FP32, scale=FP32, residual=FP32, out=FP32)
    c.x = ((c.x.float() * 16).round().clamp(-32, 32) / 16).to(t)             # 1/16 up to 2, steps of 1/64: eight bits
    c.w = ((c.w.float() * 128).round().clamp(-32, 32) / 128).to(t)           # 1/128 up to 1/4, steps of 1/512
    leaf, step = (c.x, 2.0 ** -6) if name == "x" else (c.w, 2.0 ** -9)
    leaf.requires_grad_(True)
    grad = torch.autograd.grad(c.call(), leaf, c.dy)[0]
    leaf.requires_grad_(False)
    delta, kept, ends = step * torch.sign(grad).double(), leaf.clone(), []
    for sign in (1, -1):
        leaf.copy_(kept.double() + sign * delta)
        assert torch.equal(leaf.double(), kept.double() + sign * delta)
        ends.append((c.call().double() * c.dy.double()).sum())
    leaf.copy_(kept)
    got, want = ends[0] - ends[1], (grad.double() * 2 * delta).sum()

    x, w, dy, s = c.x.double(), c.w.double(), c.dy.double(), c.scale.double()
    M, N, K = *dy.shape, x.shape[1]
    z = x @ w.T + c.bias.double()
    moved = (delta @ w.T if name == "x" else x @ delta.T).abs()
    reach = x.abs() @ w.abs().T + c.bias.double().abs() + moved
    # the ends' values: fp32 sums, the activation within 2^-20 of |z|, one rounding
    u = act64(z, act)[0]
    z_far = 2 * F32 * (K + 2) * reach
    far = 1.13 * z_far * s.abs() + (z.abs() + moved) * 2.0 ** -20 * s.abs() + 4 * F32 * ((u.abs() + 1.13 * moved) * s.abs() + c.residual.double().abs())
    # f(z + d) - f(z - d) - 2 d f'(z): d^3 / 3 times the third derivative, which is below 2
    curve = 2 / 3 * moved ** 3 * s.abs() if act else 0 * moved
    # the gradient: its slope within 2^-19, dz rounded to the operands' type, fp32 sums of its product, one rounding
    du = dy * s
    dz = du * act64(z, act)[1]
    dz_far = du.abs() * (z_far + 2.0 ** -19) + (4 * F32 + half_step(t)) * dz.abs() + half_step(t) * torch.finfo(t).tiny
    size_of, terms = ((dz.abs() + dz_far) @ w.abs(), N) if name == "x" else ((dz.abs() + dz_far).T @ x.abs(), M)
    off = dz_far @ w.abs() if name == "x" else dz_far.T @ x.abs()
    grad_far = off + 2 * F32 * (terms + 2) * size_of + half_step(t) * (grad.double().abs() + torch.finfo(t).tiny)
    slack = 2 * (far * dy.abs()).sum() + (curve * dy.abs()).sum() + (grad_far * 2 * delta.abs()).sum()
    assert (got - want).abs() <= slack, (float(got), float(want), float(slack))
    assert slack <= 0.1 * want                                              # and the bound says something
