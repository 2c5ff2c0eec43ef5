"""What linear and qkv_norm_rope promise beyond their formulas: tracing, inputs that change, huge arguments, calls from two threads."""
import threading

import pytest
import torch

from speed3r_b200 import _lib, ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16 = torch.bfloat16


@pytest.fixture(autouse=True)
def no_status():
    _lib.device_status()
    yield
    assert _lib.device_status() == 0


def compiled(f):
    ops._ops()
    torch._dynamo.reset()
    return torch.compile(f, backend="aot_eager", fullgraph=True)


def both_ways(f, inputs, n_leaves):
    results = []
    for call in (f, compiled(f)):
        leaves = [t.clone().requires_grad_(True) for t in inputs[:n_leaves]]
        outs = call(*leaves, *inputs[n_leaves:])
        sum((o.float() ** 2).sum() for o in outs).backward()
        results.append([o.detach() for o in outs] + [t.grad for t in leaves])
    return results


@pytest.mark.parametrize("K", (72, 37))
def test_compiled_linear_is_linear(K):
    g = torch.Generator(device=DEV).manual_seed(1)
    rand = lambda *s: torch.randn(*s, device=DEV, generator=g)
    inputs = [rand(2, 33, K).to(BF16), (rand(80, K) / 8).to(BF16), rand(80), rand(80), rand(2, 33, 80)]
    eager, traced = both_ways(lambda x, w, b, s, r: (ops.linear(x, w, b, "gelu", r, s), ops.linear(x, w, b)), inputs, 5)
    assert len(eager) == 7 and all(torch.equal(a, b) for a, b in zip(eager, traced))


def test_compiled_qkv_is_qkv():
    g = torch.Generator(device=DEV).manual_seed(2)
    rand = lambda *s: torch.randn(*s, device=DEV, generator=g)
    pos = torch.randint(0, 20, (2, 33, 2), device=DEV, generator=g)
    inputs = [rand(2, 33, 8 * 64).to(BF16), rand(64), rand(64), rand(64), pos, rand(20, 16), rand(20, 16)]
    f = lambda qkv, w, b, kw, pos, c, s: ops.qkv_norm_rope(qkv, 4, 2, pos, c, s, q_norm=(w, b, 1e-6), k_norm=(kw, None, 1e-5))
    eager, traced = both_ways(f, inputs, 4)
    assert len(eager) == 7 and all(torch.equal(a, b) for a, b in zip(eager, traced))


@pytest.mark.parametrize("which", ("x", "w"))
@pytest.mark.parametrize("strided", (False, True))
def test_an_operand_that_changed_in_between_is_noticed(which, strided):
    """The backward reads x and the weight again: one that was written to since is an error, also where a view of it is what the kernel reads."""
    wide = {"x": torch.randn(3, 20, 128, device=DEV).to(BF16), "w": torch.randn(40, 128, device=DEV).to(BF16)}
    x, w = (wide[n][..., :72] if strided else wide[n][..., :72].contiguous() for n in ("x", "w"))
    x.requires_grad_(True), w.requires_grad_(True)
    y = ops.linear(x, w, act="silu")
    with torch.no_grad():
        {"x": x, "w": w}[which].mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.float().sum().backward()


@pytest.mark.parametrize("act", ("gelu", "gelu_tanh", "silu"))
@pytest.mark.parametrize("M", (4, 40))
def test_huge_arguments(act, M):
    """Far out the activations are z and 0, their slopes 1 and 0, exactly."""
    x = torch.zeros(M, 16, device=DEV, dtype=BF16)
    x[:, 0] = torch.tensor([2.0 ** 60, -2.0 ** 60, 2.0 ** 30, -2.0 ** 30], device=DEV).repeat(M // 4)
    x.requires_grad_(True)
    w = torch.zeros(24, 16, device=DEV, dtype=BF16)
    w[:, 0] = 1
    y = ops.linear(x, w, torch.zeros(24, device=DEV), act=act)
    assert torch.equal(y, torch.relu(x[:, :1]).expand(M, 24))
    dx, = torch.autograd.grad(y, x, torch.ones_like(y))
    assert torch.equal(dx[:, 0], 24.0 * (x[:, 0] > 0)) and not dx[:, 1:].any()


def test_calls_from_two_threads():
    """Each on a stream of its own, with parts and without: the result of one after the other."""
    g = torch.Generator(device=DEV).manual_seed(3)
    sizes = [(64, 512, 2048), (300, 200, 136), (3, 256, 512)]
    cases = [[(torch.randn(M, K, device=DEV, generator=g).to(BF16).requires_grad_(True), (torch.randn(N, K, device=DEV, generator=g) / K ** 0.5).to(BF16)) for M, N, K in sizes]
             for _ in range(2)]
    run = lambda case: [t for x, w in case for y in [ops.linear(x, w, act="gelu")] for t in (y.detach(), *torch.autograd.grad(y, x, y.detach()))]
    want = [run(c) for c in cases]
    torch.cuda.synchronize()
    got = [None, None]

    def work(i):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(10):
                got[i] = run(cases[i])
        stream.synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert all(torch.equal(a, b) for w, o in zip(want, got) for a, b in zip(w, o))
