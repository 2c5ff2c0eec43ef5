"""Timed cases of the dense half of a block: matrix products with their epilogue, and what stands between the qkv projection and attention.

``linear``  ``ops.linear``: ``residual + act(x W^T + bias) * scale`` in bf16 or fp16, without gradients (``fwd``) or forward and
            backward (``train``)
``qkv``     ``ops.qkv_norm_rope``: the packed projection split into q, k and v, a norm of every head of q and k and their rotary
            embedding, without gradients or forward and backward

Rows are tokens: a view has 256 (224 x 224 pixels), 1008 (392 x 504) or about 1041.  The model is 1024 wide with an MLP of
4096 and 16 heads of 64; q, k, v and the gate's logits in one matrix are 3104 wide.
"""
import math

import torch

own = False

BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}
TYPE = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
DIM, MLP, QKVG = 1024, 4096, 3104


def _linear(name, mode, M, N, K, x="bf16", act="", bias="fp32", res="", scale="", out="bf16"):
    return dict(name=name, kind="linear", mode=mode, M=M, N=N, K=K, x=x, act=act, bias=bias, res=res, scale=scale, out=out)


def _qkv(name, mode, B, T, H, Hk, d, x="bf16", w="fp32", norm="layer", bias=True, axes=2, rotated=0, rows=64):
    """``rotated``: columns of a head that are rotated, 0: all of them."""
    return dict(name=name, kind="qkv", mode=mode, B=B, T=T, H=H, Hk=Hk, d=d, x=x, w=w, norm=norm, bias=bias, axes=axes, rotated=rotated or d,
                rows=rows)


def listed():
    return [
        # one token through the MLP's first matrix: latency
        _linear("linear 1 token up", "fwd", 1, MLP, DIM, act="gelu"),
        # the camera tokens of 64 views through the second one, added to the residual stream: few rows, a long sum
        _linear("linear 64 tokens down", "fwd", 64, DIM, MLP, bias="bf16", res="bf16", scale="bf16"),
        # q, k, v and the gate's logits of 8 views of 1041
        _linear("linear 8x1041 qkv+gate", "fwd", 8328, QKVG, DIM),
        # the MLP at 64 views in inference: up with its GELU; down with LayerScale, added to an fp32 residual under autocast
        _linear("linear 64x1008 up", "fwd", 64512, MLP, DIM, act="gelu"),
        _linear("linear 64x1008 down", "fwd", 64512, DIM, MLP, res="fp32", scale="fp32", out="fp32"),
        # the same in training, 2 samples of 24 views
        _linear("linear fwd+bwd 2x24x256 up", "train", 12288, MLP, DIM, act="gelu"),
        _linear("linear fwd+bwd 2x24x256 down", "train", 12288, DIM, MLP, res="fp32", scale="fp32", out="fp32"),
        # sizes that are multiples of nothing, in fp16
        _linear("linear fwd+bwd ragged", "train", 1041, 1543, 517, x="fp16", act="silu", bias="fp16", res="fp16", scale="fp16", out="fp16"),
        # one token of a stream
        _qkv("qkv 1 token", "fwd", 1, 1, 16, 16, 64),
        # frame attention of 64 views in inference
        _qkv("qkv 64x1008", "fwd", 64, 1008, 16, 16, 64),
        # frame attention in training, 2 samples of 24 views
        _qkv("qkv fwd+bwd 48x256", "train", 48, 256, 16, 16, 64),
        # a sequence rotated along one axis in half of its columns, RMS norms, heads of 80 that share keys, an odd length
        _qkv("qkv fwd+bwd 3x1041 shared heads", "train", 3, 1041, 12, 4, 80, x="fp16", w="fp16", norm="rms", bias=False, axes=1, rotated=40, rows=2048),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    mode = rng.choice(["fwd", "train"])
    x = rng.choice(["bf16", "bf16", "fp16"])
    if rng.random() < 0.6:
        N, K = (rng.choice([_log(rng, 32, 4096), 8 * _log(rng, 4, 512), 64 * _log(rng, 1, 64)]) for _ in range(2))
        M = _log(rng, 1, min(64512, 64512 * 4096 * 1024 // N // K // (1 if mode == "fwd" else 4)))
        res = rng.choice(["", "", x, "fp32"])
        case = _linear("", mode, M, N, K, x, rng.choice(["", "gelu", "gelu", "gelu_tanh", "silu"]), rng.choice(["", "fp32", x]), res,
                       rng.choice(["", "fp32", x]), res or rng.choice([x, x, "fp32"]))
    else:
        x = rng.choice([x, x, "fp32"])
        Hk = _log(rng, 1, 16)
        H = Hk * rng.choice([1, 1, 2, 4])
        d = rng.choice([64, 2 * _log(rng, 8, 128), 16 * _log(rng, 1, 16)])
        axes = rng.choice([0, 1, 2, 2, 3])
        rotated = 0 if not axes else 2 * axes * max(1, d // (2 * axes) // rng.choice([1, 1, 2]))
        rows = _log(rng, 1, max(1, min(64512, 64512 * 3 * 1024 // ((H + 2 * Hk) * d) // (1 if mode == "fwd" else 4))))
        B = min(rows, rng.choice([1, 1, 2, 3, 48]))
        norm = rng.choice(["layer", "layer", "rms", ""])
        case = _qkv("", mode, B, rows // B, H, Hk, d, x, rng.choice(["fp32", x]), norm, norm == "layer" and rng.random() < 0.8, axes, rotated,
                    rng.choice([64, 2048]))
        case["rotated"] = rotated
    del case["name"]
    return case


def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, device="cuda", generator=g).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case)
    xt = TYPE[case["x"]]
    if case["kind"] == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        # activations behind a norm, some channels stronger than others; products of about 1
        s["xt"] = (_randn(g, M, K) * (0.5 + _randn(g, K).abs())).to(xt)
        s["weight"] = (_randn(g, N, K) / math.sqrt(2 * K)).to(xt)
        s["bias_t"] = (0.1 * _randn(g, N)).to(TYPE[case["bias"]]) if case["bias"] else None
        s["scale_t"] = (0.3 * _randn(g, N)).to(TYPE[case["scale"]]) if case["scale"] else None
        # a residual stream with a few strong channels, as deep in a transformer
        s["residual"] = (_randn(g, M, N) * (0.5 + _randn(g, N).abs() ** 3)).to(TYPE[case["res"]]) if case["res"] else None
        names, made = ("xt", "weight", "bias_t", "scale_t", "residual"), (s["xt"].shape[:1] + (N,),)
        grads = [_randn(g, *made[0], dtype=TYPE[case["out"]])] if case["mode"] == "train" else None
    else:
        B, T, H, Hk, d = (case[n] for n in ("B", "T", "H", "Hk", "d"))
        wt = TYPE[case["w"]]
        s["qkv"] = (_randn(g, B, T, (H + 2 * Hk) * d) * (0.3 + _randn(g, (H + 2 * Hk) * d).abs())).to(xt)
        for n in ("q", "k"):
            s[n + "_weight"] = (1 + 0.2 * _randn(g, d)).to(wt) if case["norm"] else None
            s[n + "_bias"] = (0.1 * _randn(g, d)).to(wt) if case["bias"] else None
        s["pos"] = s["cos"] = s["sin"] = None
        if case["axes"]:
            # patches of a view in rows of about the square root, or places in a sequence; a table as the attention module keeps one
            W, rows = case["rotated"] // (2 * case["axes"]), case["rows"]
            t = torch.arange(T, device="cuda") + int(torch.randint(0, rows, (1,), device="cuda", generator=g))
            side = max(1, math.isqrt(T))
            s["pos"] = torch.stack([t // side ** i % rows for i in reversed(range(case["axes"]))], -1).expand(B, -1, -1).contiguous()
            angle = torch.outer(torch.arange(rows, device="cuda").double(), 100.0 ** (-torch.arange(W, device="cuda").double() / W))
            s["cos"], s["sin"] = angle.cos().to(xt), angle.sin().to(xt)
        names, made = ("qkv", "q_weight", "q_bias", "k_weight", "k_bias"), [(B, n, T, d) for n in (H, Hk, Hk)]
        grads = [_randn(g, *m, dtype=xt) for m in made] if case["mode"] == "train" else None
    if case["mode"] == "train":
        s["leaves"], s["grads"] = [s[n].requires_grad_(True) for n in names if s[n] is not None], grads
    return s


# ---- plain forms -----------------------------------------------------------------------------------------------------
def _plain_act(z, act):
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)))
    return z * torch.sigmoid(z) if act == "silu" else z


def _plain_linear(s):
    y = s["xt"].float() @ s["weight"].float().T
    y = y if s["bias_t"] is None else y + s["bias_t"].float()
    y = _plain_act(y, s["act"])
    y = y if s["scale_t"] is None else y * s["scale_t"].float()
    y = y if s["residual"] is None else y + s["residual"].float()
    return (y.to(TYPE[s["out"]]),)


def _plain_norm(x, weight, bias, kind, eps=1e-6):
    if not kind:
        return x
    x = x - x.mean(-1, keepdim=True) if kind == "layer" else x
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * weight.float()
    return x if bias is None else x + bias.float()


def _plain_rotate(x, s):
    if s["pos"] is None:
        return x
    B, T, heads, d = x.shape
    axes, rotated = s["axes"], s["rotated"]
    c, n = s["cos"].float()[s["pos"]][:, :, None], s["sin"].float()[s["pos"]][:, :, None]        # [B, T, 1, axes, W]
    a, b = x[..., :rotated].unflatten(-1, (axes, 2, -1)).unbind(-2)
    return torch.cat((torch.stack((a * c - b * n, b * c + a * n), -2).flatten(-3), x[..., rotated:]), -1)


def _plain_qkv(s):
    B, T, H, Hk, d = (s[n] for n in ("B", "T", "H", "Hk", "d"))
    q, k, v = s["qkv"].float().view(B, T, H + 2 * Hk, d).split((H, Hk, Hk), 2)
    q = _plain_rotate(_plain_norm(q, s["q_weight"], s["q_bias"], s["norm"]), s)
    k = _plain_rotate(_plain_norm(k, s["k_weight"], s["k_bias"], s["norm"]), s)
    return tuple(t.transpose(1, 2).to(TYPE[s["x"]]).contiguous() for t in (q, k, v))


def run(s):
    with torch.set_grad_enabled(s["mode"] == "train"):
        if own:
            from speed3r_b200 import ops
            if s["kind"] == "linear":
                out = (ops.linear(s["xt"], s["weight"], s["bias_t"], s["act"] or None, s["residual"], s["scale_t"], TYPE[s["out"]]),)
            else:
                q_norm, k_norm = ((s[n + "_weight"], s[n + "_bias"], 1e-6) if s["norm"] else None for n in ("q", "k"))
                out = ops.qkv_norm_rope(s["qkv"], s["H"], s["Hk"], s["pos"], s["cos"], s["sin"], q_norm, k_norm, s["norm"] or "layer")
        else:
            out = _plain_linear(s) if s["kind"] == "linear" else _plain_qkv(s)
    if s["mode"] == "fwd":
        return out
    return tuple(t.detach() for t in out) + torch.autograd.grad(out, s["leaves"], s["grads"])


# ---- what a pass cannot do without -----------------------------------------------------------------------------------
def work(case):
    x = BYTES[case["x"]]
    if case["kind"] == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        small = N * sum(BYTES[case[n]] for n in ("bias", "scale") if case[n])
        res, out = BYTES[case["res"]] if case["res"] else 0, BYTES[case["out"]]
        total, flops = M * K * x + N * K * x + M * N * (res + out) + small, 2 * M * N * K
        if case["mode"] == "train":                      # dy in, dx, dW and what else has a gradient out
            total, flops = total + M * N * (out + res) + M * K * x + N * K * x + small, 3 * flops
        return {"bytes": total, "flops": flops}
    n = case["B"] * case["T"] * (case["H"] + 2 * case["Hk"]) * case["d"]
    pos = case["B"] * case["T"] * case["axes"] * 8
    # q, k, v in and out; backward: their gradients in and out
    return {"bytes": n * x * (2 if case["mode"] == "fwd" else 4) + pos, "flops": n * (12 if case["mode"] == "fwd" else 40)}


# ---- the definition in 64 bits ---------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return _exact_linear(s) if case["kind"] == "linear" else _exact_qkv(s)


def _exact_act(z, act):
    """(act(z), its derivative)"""
    if act == "gelu":
        below = torch.special.ndtr(z)
        return z * below, below + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if act == "gelu_tanh":
        w = 2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)
        p = 1 / (1 + torch.exp(-w))
        return z * p, p + z * p * (1 - p) * 2 * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * z * z)
    if act == "silu":
        p = 1 / (1 + torch.exp(-z))
        return z * p, p * (1 + z * (1 - p))
    return z, torch.ones_like(z)


def _exact_linear(s):
    x, w = s["xt"].double(), s["weight"].double()
    z = torch.einsum("mk,nk->mn", x, w)
    if s["bias_t"] is not None:
        z += s["bias_t"].double()
    u, slope = _exact_act(z, s["act"])
    del z
    c = 1.0 if s["scale_t"] is None else s["scale_t"].double()
    y = u * c + (0 if s["residual"] is None else s["residual"].double())
    if s["mode"] == "fwd":
        return (y,)
    dy = s["grads"][0].double()
    dz = dy * c * slope
    out = [y, torch.einsum("mn,nk->mk", dz, w), torch.einsum("mn,mk->nk", dz, x)]
    if s["bias_t"] is not None:
        out.append(dz.sum(0))
    if s["scale_t"] is not None:
        out.append((dy * u).sum(0))
    if s["residual"] is not None:
        out.append(dy)
    return tuple(out)


def _exact_matrix(s):
    """What rotation multiplies a token's pairs with, as complex numbers [B, T, 1, pairs]; pair i of axis a lies W apart."""
    c, n = (t.double()[s["pos"]].flatten(2) for t in (s["cos"], s["sin"]))
    return torch.complex(c, n)[:, :, None]


def _exact_pairs(s):
    """Columns of the first and of the second members."""
    W = s["rotated"] // (2 * s["axes"])
    first = torch.tensor([2 * W * a + i for a in range(s["axes"]) for i in range(W)], device="cuda")
    return first, first + W


def _exact_qkv(s):
    B, T, H, Hk, d = (s[n] for n in ("B", "T", "H", "Hk", "d"))
    x = s["qkv"].double().view(B, T, H + 2 * Hk, d)
    outs, grads, back = [], [], []
    turn = _exact_matrix(s) if s["axes"] else None
    first, second = _exact_pairs(s) if s["axes"] else (None, None)

    def rotate(t, by):
        if turn is None:
            return t
        t = t.clone()
        z = torch.complex(t[..., first], t[..., second]) * by
        t[..., first], t[..., second] = z.real, z.imag
        return t

    start = 0
    for i, (n, heads) in enumerate((("q", H), ("k", Hk), ("v", Hk))):
        t = x[:, :, start:start + heads]
        start += heads
        dt = s["grads"][i].double().transpose(1, 2) if s["mode"] == "train" else None
        if n == "v":
            outs.append(t)
            back.append(dt)
            continue
        w, b = s[n + "_weight"], s[n + "_bias"]
        centre, inv, unit = 0.0, 1.0, t
        if s["norm"]:
            centre = t.mean(-1, keepdim=True) if s["norm"] == "layer" else 0.0
            inv = (((t - centre) ** 2).sum(-1, keepdim=True) / d + 1e-6) ** -0.5
            unit = (t - centre) * inv
        h = unit if w is None else unit * w.double()
        outs.append(rotate(h if b is None else h + b.double(), turn))
        if dt is None:
            continue
        dh = rotate(dt, None if turn is None else turn.conj())
        if s["norm"]:
            grads.append((dh * unit).sum((0, 1, 2)))
            if b is not None:
                grads.append(dh.sum((0, 1, 2)))
            e = dh * w.double()
            dh = e - unit * (e * unit).sum(-1, keepdim=True) / d
            dh = inv * (dh - e.sum(-1, keepdim=True) / d if s["norm"] == "layer" else dh)
        back.append(dh)
    outs = [t.transpose(1, 2).contiguous() for t in outs]
    return tuple(outs) if s["mode"] == "fwd" else tuple(outs) + (torch.cat(back, 2).reshape(B, T, -1),) + tuple(grads)
