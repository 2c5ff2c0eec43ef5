"""Timed cases of the operators around the sparse attention: a block's norms, its 8-bit projections, its optimiser.

``norm``    ``ops.residual_norm``: residual + gate * LayerScale * branch, and the norm of the sum; without gradients
            (``fwd``), forward and backward (``train``), or with the norm's result as 8-bit tokens (``int8``,
            ``ops.residual_norm_int8``)
``linear``  ``ops.int8_linear`` on tokens that ``ops.quantize_tokens`` makes of bf16 activations within the call, or
            (``given``) on tokens that are 8-bit already
``adamw``   ``ops.adamw_step`` over a list of tensors, with ``ops.grad_norm`` in front where gradients are clipped and
            ``ops.adamw_state`` behind it where the state is held in 8 bits

Rows are tokens: a view has 256 (224 x 224 pixels), 1008 (392 x 504) or about 1041.  The model is 1024 wide with an MLP of
4096; q, k, v and the gate's logits in one matrix are 3104 wide.
"""
import math

import torch

own = False

BLOCK = 256          # elements of an 8-bit state that share an exponent
BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}
TYPE = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
DIM, MLP, QKVG = 1024, 4096, 3104

# tensors of one block: q, k, v and gate; projection; MLP; two norms and LayerScales; norms of q and k
LAYER = [(QKVG, DIM), (QKVG,), (DIM, DIM), (DIM,), (MLP, DIM), (MLP,), (DIM, MLP), (DIM,)] + 6 * [(DIM,)] + 4 * [(64,)]


def listed():
    return [
        # one token of a stream: latency
        dict(name="norm fwd 1 token", kind="norm", mode="fwd", B=1, T=1, C=1024, x="bf16", y="bf16", h="bf16", w="bf16", norm="layer",
             scale=True, gate="", post=False),
        # attention to MLP of one block in inference at 64 views: fp32 residual under autocast
        dict(name="norm fwd 64x1008", kind="norm", mode="fwd", B=1, T=64512, C=1024, x="fp32", y="bf16", h="bf16", w="fp32", norm="layer",
             scale=True, gate="", post=False),
        # the same in front of an 8-bit product, 8 views of 1041
        dict(name="norm int8 8x1041", kind="norm", mode="int8", B=1, T=8328, C=1024, x="bf16", y="bf16", h="bf16", w="bf16", norm="layer",
             scale=True, gate="", post=False),
        # training: 2 samples of 24 views, LayerScale, stochastic depth (a factor per sample)
        dict(name="norm fwd+bwd 2x24x256", kind="norm", mode="train", B=2, T=6144, C=1024, x="fp32", y="bf16", h="bf16", w="fp32",
             norm="layer", scale=True, gate="sample", post=False),
        # norms on both sides of a block, a gate per sample and channel, odd width and length, all bf16
        dict(name="norm fwd+bwd sandwich 3x1041", kind="norm", mode="train", B=3, T=1041, C=1540, x="bf16", y="bf16", h="bf16", w="bf16",
             norm="rms", scale=False, gate="channel", post=True),
        # one token through the MLP's first matrix
        dict(name="linear 1 token", kind="linear", M=1, N=4096, K=1024, given=False, bias=True, out="bf16"),
        # q, k, v and the gate's logits of 8 views of 1041
        dict(name="linear 8x1041 qkv+gate", kind="linear", M=8328, N=3104, K=1024, given=True, bias=True, out="bf16"),
        # the MLP's second matrix at 64 views, activations in bf16
        dict(name="linear 64x1008 down", kind="linear", M=64512, N=1024, K=4096, given=False, bias=True, out="bf16"),
        # the MLP's first matrix at 64 views
        dict(name="linear 64x1008 up", kind="linear", M=64512, N=4096, K=1024, given=True, bias=True, out="bf16"),
        # what is left to train when matrices are frozen: norms, LayerScales and biases of one block, odd sizes among them
        dict(name="adamw vectors", kind="adamw", shapes="vectors", layers=1, bits=32, p="fp32", clip=False, seed=-1),
        # one block, clipped
        dict(name="adamw 1 block", kind="adamw", shapes="layer", layers=1, bits=32, p="fp32", clip=True, seed=-1),
        # the 18 blocks of the decoder with 8-bit states, stochastic rounding, clipped
        dict(name="adamw 18 blocks 8-bit", kind="adamw", shapes="layer", layers=18, bits=8, p="fp32", clip=True, seed=11),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm", "norm", "norm", "linear", "linear", "adamw", "adamw"])
    if kind == "norm":
        mode = rng.choice(["fwd", "train", "train", "int8"])
        C = rng.choice([_log(rng, 64, 4096), 8 * _log(rng, 8, 512), 8 * _log(rng, 8, 512)])
        rows = _log(rng, 1, min(64512, 64512 * 1024 // C // (1 if mode == "fwd" else 4)))
        B = min(rows, rng.choice([1, 1, 2, 3, 16]))
        x = rng.choice(["fp32", "bf16", "fp16"])
        y = x if x == "fp16" else rng.choice(["bf16", x])
        return dict(kind=kind, mode=mode, B=B, T=rows // B, C=C, x=x, y=y, h="bf16" if mode == "int8" else y, w=rng.choice(["fp32", y]),
                    norm=rng.choice(["layer", "rms"]), scale=rng.random() < 0.7, gate=rng.choice(["", "", "sample", "token", "channel"]), post=rng.random() < 0.3)
    if kind == "linear":
        N, K = (rng.choice([_log(rng, 64, 4096), 16 * _log(rng, 4, 256)]) for _ in range(2))
        return dict(kind=kind, M=_log(rng, 1, min(64512, 64512 * 4096 * 1024 // N // K)), N=N, K=K, given=rng.random() < 0.5,
                    bias=rng.random() < 0.7, out=rng.choice(["bf16", "bf16", "fp16", "fp32"]))
    bits = rng.choice([8, 8, 32])
    return dict(kind=kind, shapes=rng.choice(["vectors", "layer", "ragged"]), layers=_log(rng, 1, 18), bits=bits, p=rng.choice(["fp32", "bf16"]),
                clip=rng.random() < 0.6, seed=rng.choice([-1, rng.randrange(1 << 30)]))


def _shapes(case):
    if case["shapes"] == "vectors":
        one = [s for s in LAYER if len(s) == 1] + [(1,), (333,), (1041,)]
    elif case["shapes"] == "layer":
        one = LAYER
    else:                                    # widths that are multiples of nothing
        one = [(1041, 331), (331,), (77, 1041), (5,), (3, 3, 61), (1,), (2049,), (255,), (257,)]
    return one * case["layers"]


def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, device="cuda", generator=g).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case)
    if case["kind"] == "norm":
        B, T, C = case["B"], case["T"], case["C"]
        wt = TYPE[case["w"]]
        # a residual stream with a few strong channels, as deep in a transformer
        s["xt"] = (_randn(g, B, T, C) * (0.5 + _randn(g, C).abs() ** 3)).to(TYPE[case["x"]])
        s["yt"] = _randn(g, B, T, C, dtype=TYPE[case["y"]])
        s["weight"], s["bias"] = (1 + 0.2 * _randn(g, C)).to(wt), (0.1 * _randn(g, C)).to(wt) if case["norm"] == "layer" else None
        s["post_weight"] = (1 + 0.2 * _randn(g, C)).to(wt) if case["post"] else None
        s["post_bias"] = (0.1 * _randn(g, C)).to(wt) if case["post"] and case["norm"] == "layer" else None
        s["scale_t"] = (0.3 * _randn(g, C)).to(wt) if case["scale"] else None
        s["gate_t"] = None
        if case["gate"] == "sample":                     # stochastic depth: some branches are left out, the rest scaled up
            s["gate_t"] = ((torch.rand(B, 1, 1, device="cuda", generator=g) < 0.8).float() / 0.8).to(wt)
        elif case["gate"]:
            s["gate_t"] = (0.5 * _randn(g, *((B, T, 1) if case["gate"] == "token" else (B, 1, C)))).to(wt)
        if case["mode"] == "train":
            names = [n for n in ("xt", "yt", "weight", "bias", "scale_t", "gate_t", "post_weight", "post_bias") if s[n] is not None]
            if case["gate"] == "sample":
                names.remove("gate_t")                   # drawn, not learnt
            s["leaves"] = [s[n].requires_grad_(True) for n in names]
            s["dr"], s["dh"] = 0.1 * _randn(g, B, T, C), _randn(g, B, T, C)
            s["dr"], s["dh"] = s["dr"].to(TYPE[case["x"]]), s["dh"].to(TYPE[case["h"]])
    elif case["kind"] == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        x = (_randn(g, M, K) * (0.5 + _randn(g, K).abs())).bfloat16()
        w = 0.02 * _randn(g, N, K)
        s["x"] = x
        if case["given"]:
            s["x"], s["xs"] = _plain_quantize(x)
        s["wq"], s["ws"] = _plain_quantize(w)
        s["bias_t"] = 0.1 * _randn(g, N) if case["bias"] else None
    else:
        shapes = _shapes(case)
        size = [math.prod(x) for x in shapes]
        room = torch.tensor([x + -x % BLOCK for x in size], device="cuda")
        n, pt = int(room.sum()), TYPE[case["p"]]
        # parameters, gradients and states lie in one buffer each, every tensor in whole blocks; what fills a block up is zero
        first = torch.repeat_interleave(room.cumsum(0) - room, room)
        used = torch.arange(n, device="cuda") - first < torch.repeat_interleave(torch.tensor(size, device="cuda"), room)
        # heavy tails: an element's gradients have a size of their own, and so has a tensor's
        spread = torch.exp(1.5 * _randn(g, n)) * torch.exp(_randn(g, len(size))).repeat_interleave(room) * 1e-3 * used
        s["g"], s["p_"] = (_randn(g, n) * spread).to(pt), (0.02 * _randn(g, n) * used).to(pt)
        s["m"], s["v"] = _randn(g, n) * spread * 0.3, (0.5 + torch.rand(n, device="cuda", generator=g)) * spread * spread
        s["scales"] = None
        if case["bits"] == 8:
            (s["m"], me), (s["v"], ve) = _encode(s["m"], 4, True, None), _encode(s["v"], 5, False, None)
            s["e"] = torch.stack((me, ve))
            s["scales"] = list(s["e"].split((room // BLOCK).tolist(), 1))
            s["m_value"], s["v_value"] = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
            s["values"] = _views(s["m_value"], shapes), _views(s["v_value"], shapes)
        s["params"], s["grads"], s["exp_avg"], s["exp_avg_sq"] = (_views(s[x], shapes) for x in ("p_", "g", "m", "v"))
        s["step"] = torch.tensor(20, device="cuda")
    return s


def _views(flat, shapes):
    """The tensors that lie in ``flat``, each from the start of a block on."""
    size = [math.prod(x) for x in shapes]
    return [t[:n].view(x) for t, n, x in zip(flat.split([n + -n % BLOCK for n in size]), size, shapes)]


# ---- plain forms -----------------------------------------------------------------------------------------------------
def _plain_norm(x, weight, bias, kind, eps=1e-6):
    x = x - x.mean(-1, keepdim=True) if kind == "layer" else x
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps)
    x = x if weight is None else x * weight.float()
    return x if bias is None else x + bias.float()


def _plain_residual_norm(s):
    u = s["yt"].float()
    if s["post"]:
        u = _plain_norm(u, s["post_weight"], s["post_bias"], s["norm"])
    if s["scale_t"] is not None:
        u = u * s["scale_t"].float()
    if s["gate_t"] is not None:
        u = u * s["gate_t"].float()
    r = s["xt"].float() + u
    # the sum as it is stored, in 32 bits, so that its gradient is rounded once, at the end
    r = r + (r.to(TYPE[s["x"]]).float() - r).detach()
    return r.to(TYPE[s["x"]]), _plain_norm(r, s["weight"], s["bias"], s["norm"])


def _plain_quantize(x):
    x = x.float()
    big = x.abs().amax(-1)
    q = torch.where(big[..., None] > 0, x * (127 / big)[..., None], 0).round()
    return q.to(torch.int8), big / 127


def _encode(x, exponent_bits, signed, dither):
    """Codes of sign, exponent and three bits of mantissa, and the exponent of each block: 2^(e - 127) times the largest code,
    1.875, is at least the block's largest magnitude.  ``dither``: what is added below the last bit that is kept, None: to nearest."""
    blocks = x.view(-1, BLOCK)
    e = ((blocks.abs().view(torch.int32).amax(1).clamp(max=0x7F800000) + 0xFFFFF) >> 23).clamp(min=27)
    e = torch.where(e > 227, 255, e)
    y = blocks.abs() * ((254 - e) << 23).view(torch.float32)[:, None] * 2.0 ** (2 ** exponent_bits - 128)
    bits = y.view(torch.int32)
    u = 0x7FFFF + (bits >> 20 & 1) if dither is None else dither.view(-1, BLOCK)
    code = (bits + u >> 20).clamp(max=2 ** (exponent_bits + 3) - 1)
    if signed:
        code = code | (blocks < 0).int() << 7
    else:
        code = torch.maximum(code, (blocks > 0).int())
    return code.to(torch.uint8).view(-1), e.to(torch.uint8)


def _decode(code, e, exponent_bits, signed):
    c = code.view(-1, BLOCK).int()
    value = ((c & 127 if signed else c) << 20).view(torch.float32) * 2.0 ** (128 - 2 ** exponent_bits)
    value = value * (e.int() << 23).view(torch.float32)[:, None]
    value = torch.where(e[:, None] == 255, math.nan, value)
    return (torch.where(c > 127, -value, value) if signed else value).view(-1)


def _round_of(a, c, k, seven):
    """One of ``seven`` rounds of Philox 2x32 and the rounds behind it: (a, c) -> (hi(M a) ^ k ^ c, lo(M a))."""
    m = a * 0xD256D193
    a, c = (m >> 32 & 0xFFFFFFFF) ^ k ^ c, m & 0xFFFFFFFF
    return (a, c) if seven == 1 else _round_of(a, c, k + 0x9E3779B9 & 0xFFFFFFFF, seven - 1)


def _dither(tensors, step, seed):
    """32 random bits for every element: its pair within the tensor and the step are the counter, seed and tensor the key."""
    pairs = [(t.numel() + -t.numel() % BLOCK) // 2 for t in tensors]
    pair = torch.cat([torch.arange(n, device="cuda") for n in pairs])
    key = torch.cat([torch.full((n,), seed + i * 0x85EBCA6B & 0xFFFFFFFF, device="cuda") for i, n in enumerate(pairs)])
    return torch.stack(_round_of(pair, step.expand(pair.shape), key, 7), -1).view(-1)


def _plain_adamw(s, lr=1e-3, b1=0.9, b2=0.999, eps=1e-8, decay=0.05, max_norm=1.0):
    eight, g, norm = s["bits"] == 8, s["g"].float(), None
    if s["clip"]:
        norm = (g.double() ** 2).sum().sqrt().float()
        g = g * torch.clamp(max_norm / (norm + 1e-6), max=1.0)
    step = s["step"].add_(1)
    m, v = s["m"], s["v"]
    if eight:
        m, v = _decode(m, s["e"][0], 4, True), _decode(v, s["e"][1], 5, False)
    m = m * b1 + g * (1 - b1)
    v = v * b2 + g * g * (1 - b2)
    t = step.double()
    size_of_step, root = (lr / (1 - b1 ** t)).float(), torch.sqrt(1 - b2 ** t).float()
    p = s["p_"].float() * (1 - lr * decay) - size_of_step * (m / (torch.sqrt(v) / root + eps))
    low = None if s["seed"] < 0 else _dither(s["params"], step, s["seed"])
    if s["p"] == "bf16" and low is not None:
        p = ((p.view(torch.int32) + ((low >> 22) * 64 + 32).int()) >> 16 << 16).view(torch.float32)
    s["p_"].copy_(p)
    if eight:
        mc, me = _encode(m, 4, True, None if low is None else ((low & 0xFF) << 12 | 0x800).int())
        vc, ve = _encode(v, 5, False, None if low is None else ((low >> 8 & 0x3FFF) << 6 | 0x20).int())
        s["m"].copy_(mc), s["v"].copy_(vc), s["e"].copy_(torch.stack((me, ve)))
        s["m_value"].copy_(_decode(mc, me, 4, True)), s["v_value"].copy_(_decode(vc, ve, 5, False))
    else:
        s["m"].copy_(m), s["v"].copy_(v)
    return _adamw_outputs(s, norm)


def _adamw_outputs(s, norm):
    names = ("p_", "m_value", "v_value") if s["bits"] == 8 else ("p_", "m", "v")
    return tuple(s[n] for n in names) + (() if norm is None else (norm,))


def run(s):
    if own:
        from speed3r_b200 import ops
    if s["kind"] == "norm":
        norm = (s["weight"], s["bias"], 1e-6)
        post = (s["post_weight"], s["post_bias"], 1e-6) if s["post"] else None
        if s["mode"] == "int8":
            if own:
                r, q, qs = ops.residual_norm_int8(s["xt"], s["yt"], norm, s["scale_t"], s["gate_t"], post, s["norm"])
            else:
                r, h = _plain_residual_norm(s)
                q, qs = _plain_quantize(h)
            return r, (q * qs[..., None]).to(TYPE[s["h"]]), qs
        if own:
            with torch.set_grad_enabled(s["mode"] == "train"):
                r, h = ops.residual_norm(s["xt"], s["yt"], norm, s["scale_t"], s["gate_t"], post, s["norm"], TYPE[s["h"]])
        else:
            with torch.set_grad_enabled(s["mode"] == "train"):
                r, h = _plain_residual_norm(s)
                h = h.to(TYPE[s["h"]])
        if s["mode"] == "fwd":
            return r, h
        return (r.detach(), h.detach()) + torch.autograd.grad((r, h), s["leaves"], (s["dr"], s["dh"]))
    if s["kind"] == "linear":
        if own:
            q, qs = (s["x"], s["xs"]) if s["given"] else ops.quantize_tokens(s["x"])
            return ops.int8_linear(q, qs, s["wq"], s["ws"], s["bias_t"], TYPE[s["out"]])
        q, qs = (s["x"], s["xs"]) if s["given"] else _plain_quantize(s["x"])
        # sums of products of 8-bit numbers pass 2^24: in 64 bits they are exact
        y = (q.double() @ s["wq"].double().T).float() * qs[:, None] * s["ws"]
        return (y if s["bias_t"] is None else y + s["bias_t"]).to(TYPE[s["out"]])
    if own:
        norm = ops.grad_norm(s["grads"]) if s["clip"] else None
        ops.adamw_step(s["params"], s["grads"], s["exp_avg"], s["exp_avg_sq"], s["step"], lr=1e-3, betas=(0.9, 0.999), eps=1e-8,
                       weight_decay=0.05, grad_norm=norm, max_norm=1.0 if s["clip"] else None, scales=s["scales"],
                       seed=None if s["seed"] < 0 else s["seed"])
        if s["bits"] == 8:
            ops.adamw_state(s["exp_avg"], s["exp_avg_sq"], s["scales"], out=s["values"])
        return _adamw_outputs(s, norm)
    return _plain_adamw(s)


# ---- what a pass cannot do without -----------------------------------------------------------------------------------
def work(case):
    if case["kind"] == "norm":
        n, b = case["B"] * case["T"] * case["C"], BYTES
        per = 2 * b[case["x"]] + b[case["y"]] + (1 if case["mode"] == "int8" else b[case["h"]])          # x, y in; r, h out
        if case["mode"] == "train":
            per += 2 * b[case["x"]] + b[case["y"]] + b[case["h"]]                                        # dr, dh in; dx, dy out
        return {"bytes": n * per, "flops": n * (40 if case["mode"] == "train" else 12)}
    if case["kind"] == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        return {"bytes": M * K * (1 if case["given"] else 2) + N * K + M * N * BYTES[case["out"]] + 4 * (M + 2 * N), "flops": 2 * M * N * K}
    n, b = sum(math.prod(x) for x in _shapes(case)), BYTES[case["p"]]
    return {"bytes": n * (3 * b + (16 if case["bits"] == 32 else 4 + 8)), "flops": n * 20}


# ---- the definition in 64 bits ---------------------------------------------------------------------------------------
def exact(case, seed):
    if case["kind"] == "adamw":
        return None if sum(math.prod(x) for x in _shapes(case)) > 60e6 else _exact_adamw(prepare(case, seed))
    s = prepare(case, seed)
    if case["kind"] == "norm":
        with torch.no_grad():
            return _exact_norm(s)
    M, N, K = case["M"], case["N"], case["K"]
    if M * N > 300e6 or M * K > 300e6:
        return None
    q, qs = (s["x"], s["xs"].double()) if case["given"] else _exact_quantize(s["x"].double())
    y = (torch.einsum("mk,nk->mn", q.double(), s["wq"].double()) * qs[:, None]) * s["ws"].double()[None]
    return y + (0 if s["bias_t"] is None else s["bias_t"].double())


def _exact_quantize(x):
    big = x.abs().max(-1).values
    q = torch.round(x * torch.where(big == 0, 0, 127 / big).unsqueeze(-1))
    return q, big / 127


def _statistics(x, kind, eps):
    """(normalised x, factor) of every row."""
    mean = x.sum(-1, keepdim=True) / x.shape[-1] if kind == "layer" else torch.zeros_like(x[..., :1])
    factor = 1 / torch.sqrt(((x - mean) ** 2).sum(-1, keepdim=True) / x.shape[-1] + eps)
    return (x - mean) * factor, factor


def _through(d, n, factor, kind):
    """Gradient with respect to what was normalised to n, from the gradient d of n."""
    along = n * (d * n).sum(-1, keepdim=True) / n.shape[-1]
    return factor * (d - along - (d.sum(-1, keepdim=True) / n.shape[-1] if kind == "layer" else 0))


def _exact_norm(s):
    kind, one = s["norm"], torch.ones((), dtype=torch.float64, device="cuda")
    of = lambda t, other: other if t is None else t.detach().double()                            # noqa: E731
    x, y = of(s["xt"], None), of(s["yt"], None)
    w, b, c, gate, pw, pb = (of(s[n], o) for n, o in (("weight", one), ("bias", 0 * one), ("scale_t", one), ("gate_t", one),
                                                      ("post_weight", one), ("post_bias", 0 * one)))
    ny, fy = _statistics(y, kind, 1e-6) if s["post"] else (y, None)
    u = ny * pw + pb if s["post"] else y
    r = x + u * c * gate
    nr, fr = _statistics(r.to(TYPE[s["x"]]).double(), kind, 1e-6)
    h = nr * w + b
    if s["mode"] == "fwd":
        return r, h
    if s["mode"] == "int8":
        q, qs = _exact_quantize(h)
        return r, q * qs[..., None], qs
    dr, dh = s["dr"].double(), s["dh"].double()
    G = dr + _through(dh * w, nr, fr, kind)
    du = G * c * gate
    dy = _through(du * pw, ny, fy, kind) if s["post"] else du
    rows = lambda t: t.flatten(0, 1).sum(0)                                                      # noqa: E731
    out = [r, h, G, dy, rows(dh * nr)]
    if s["bias"] is not None:
        out.append(rows(dh))
    if s["scale_t"] is not None:
        out.append(rows(G * gate * u))
    if s["gate"] in ("token", "channel"):
        out.append((G * c * u).sum(1 if s["gate"] == "channel" else 2, keepdim=True))
    if s["post"]:
        out.append(rows(du * ny))
        if s["post_bias"] is not None:
            out.append(rows(du))
    return tuple(out)


def _exact_code(x, exponent_bits, random_bits, random):
    """x rounded to what blocks of codes hold, in 64 bits; ``random``: integers of ``random_bits`` bits, or None."""
    x = torch.nn.functional.pad(x, (0, -x.numel() % BLOCK)).view(-1, BLOCK)
    big = x.abs().amax(1, keepdim=True)
    # the smallest power of two whose 1.875-fold reaches the largest magnitude
    unit = torch.exp2(torch.ceil(torch.log2(big / 1.875)).clamp(-100, 100))
    unit = torch.where(unit * 1.875 < big, unit * 2, torch.where(unit * 0.9375 >= big, unit / 2, unit)).clamp(min=2.0 ** -100)
    z = x.abs() / unit
    bottom = 2 - 2 ** exponent_bits                                    # exponent of the smallest normal number
    last = torch.exp2(torch.floor(torch.log2(z.clamp(min=2.0 ** -60))).clamp(min=bottom) - 3)
    if random is None:
        z = torch.round(z / last) * last
    else:
        z = torch.floor(z / last + (random.view(-1, BLOCK).double() + 0.5) / 2 ** random_bits) * last
    z = z.clamp(max=1.875)
    if exponent_bits == 5:
        z = torch.where(x > 0, z.clamp(min=2.0 ** (bottom - 3)), z)
    return (torch.sign(x) * z * unit).view(-1)


def _exact_values(code, e, exponent_bits):
    """What codes stand for: (1 + f / 8) 2^(E - largest E), and f / 8 where E is 0."""
    code = torch.nn.functional.pad(code.reshape(-1), (0, -code.numel() % BLOCK)).long().view(-1, BLOCK)
    sign = torch.where((code >= 128) & (exponent_bits == 4), -1.0, 1.0)
    code = code % (8 << exponent_bits)
    E, f, top = code // 8, (code % 8).double() / 8, 2 ** exponent_bits - 1
    value = torch.where(E > 0, (1 + f) * torch.exp2((E - top).double()), f * 2.0 ** (1 - top))
    return (sign * value * torch.exp2(e.double() - 127)[:, None]).view(-1)


def _exact_random(n, step, key):
    a, c = torch.arange((n + -n % BLOCK) // 2, device="cuda"), torch.tensor(step, device="cuda")
    for i in range(7):
        low, high = (a & 0xFFFF) * 0xD256D193, (a >> 16) * 0xD256D193            # in two halves: no product passes 63 bits
        whole_low = (low + ((high & 0xFFFF) << 16)) & 0xFFFFFFFF
        whole_high = (high + (low >> 16)) >> 16
        a, c = whole_high & 0xFFFFFFFF ^ (key + i * 0x9E3779B9) % 2 ** 32 ^ c, whole_low
    return torch.stack((a, c), 1).view(-1)


def _exact_adamw(s):
    t = int(s["step"]) + 1
    total = math.sqrt(sum(float((g.double() ** 2).sum()) for g in s["grads"]))
    factor = min(1.0, 1.0 / (total + 1e-6)) if s["clip"] else 1.0
    params, first, second = [], [], []
    for i, (p, g) in enumerate(zip(s["params"], s["grads"])):
        n, g = p.numel(), g.double().view(-1) * factor
        m, v = s["exp_avg"][i], s["exp_avg_sq"][i]
        if s["bits"] == 8:
            m, v = _exact_values(m, s["scales"][i][0], 4)[:n], _exact_values(v, s["scales"][i][1], 5)[:n]
        m, v = 0.9 * m.double().view(-1) + 0.1 * g, 0.999 * v.double().view(-1) + 0.001 * g * g
        q = p.double().view(-1) * (1 - 1e-3 * 0.05) - 1e-3 / (1 - 0.9 ** t) * m / (torch.sqrt(v / (1 - 0.999 ** t)) + 1e-8)
        if s["bits"] == 8:
            low = None if s["seed"] < 0 else _exact_random(n, t, (s["seed"] + i * 0x85EBCA6B) % 2 ** 32)
            m = _exact_code(m, 4, 8, None if low is None else low & 0xFF)[:n]
            v = _exact_code(v, 5, 14, None if low is None else low >> 8 & 0x3FFF)[:n]
        params.append(q), first.append(m), second.append(v)
    whole = lambda ts: torch.cat([torch.nn.functional.pad(t, (0, -t.numel() % BLOCK)) for t in ts])  # noqa: E731
    return (whole(params), whole(first), whole(second)) + ((torch.tensor(total, dtype=torch.float64),) if s["clip"] else ())
