"""The package's operators over the C-ABI kernels.

Public functions mirror the reference's op signatures:

* ``flash_attn_topk_func(q_c, k_c, v_c, topk_val, bias=None, causal=False, softmax_scale=None)``
  -> ``(o_c, idx)``      (pi3/models/sparse_attn/flash_attention_topk.py:633-668)
* ``topk_blocksparse_attention(q, k, v, topk_idx, block_size, softmax_scale=None)`` -> ``o``
  (pi3/models/sparse_attn/topk_blocksparse_attention.py:1093-1121)

the rest of a block around them (``residual_norm``), its projections in 8 bits (``quantize_tokens``, ``int8_linear``) and the step
that ends a training iteration (``grad_norm``, ``adamw_step``), plus the pieces the reference leaves to eager PyTorch (sparse_attention.py:97-102, 127-136):

* ``pool_tokens(x, kernel, stride)``: mean pooling along the sequence
* ``sel_attn_merge(q, k, v, idx, gate, o_c, block_size)``: selection attention with the gated
  merge fused, returning ``[B,T,H*d]``

Allocation, argument checks and autograd wiring are native (``csrc/torch/bindings.cpp``, a ``torch.library``
namespace over the C ABI); this file holds the Python signatures and the shape functions for
``torch.compile``.  CPU tensors, types that an operator does not take (the attention's take bf16, the operators around it fp32 and
fp16 too) and a missing library raise: there is no fallback.
"""
from __future__ import annotations

import math
import threading
from typing import Optional, Tuple

import torch
from torch import Tensor

from . import _lib

_BF16 = torch.bfloat16
_lock = threading.Lock()
_ns = None


def _register_fakes() -> None:
    fake = torch.library.register_fake

    @fake("speed3r_b200::pool_fwd")
    def _(x, kernel, stride):
        B, H, T, d = x.shape
        return x.new_empty(B, H, (T - kernel) // stride + 1, d)

    @fake("speed3r_b200::pool_bwd")
    def _(d_out, T, kernel, stride):
        B, H, Nc, d = d_out.shape
        return d_out.new_empty(B, H, T, d)

    def cmp_fwd(q_c, k_c, v_c, topk, scale, group=0, take=0):
        B, H, Nq, d = q_c.shape
        return (q_c.new_empty(B, H, Nq, d), q_c.new_empty(B, H, Nq, dtype=torch.float32),
                q_c.new_empty(B, H, Nq, topk, dtype=torch.int32))

    fake("speed3r_b200::cmp_attn_topk_fwd", cmp_fwd)
    fake("speed3r_b200::cmp_attn_blocktopk_fwd", cmp_fwd)

    @fake("speed3r_b200::cmp_attn_bwd")
    def _(q_c, k_c, v_c, o_c, lse, do_c, scale):
        return tuple(t.new_empty(t.shape) for t in (q_c, k_c, v_c))

    @fake("speed3r_b200::sel_attn_fwd")
    def _(q, k, v, idx, gate, o_c, block, scale, want_o, want_lse, kv_chunks):
        B, H, Tq, d = q.shape
        return (q.new_empty(B, H, Tq, d) if want_o else q.new_empty(0),
                q.new_empty(B, H, Tq, dtype=torch.float32) if want_lse else q.new_empty(0, dtype=torch.float32),
                q.new_empty(B, Tq, H * d) if gate is not None else q.new_empty(0))

    @fake("speed3r_b200::build_key_csr")
    def _(idx, num_key_blocks):
        B, H, Nq, K = idx.shape
        return idx.new_empty(B, H, num_key_blocks + 1), idx.new_empty(B, H, Nq * K)

    @fake("speed3r_b200::sel_attn_bwd")
    def _(q, k, v, idx, lse, delta, do_s, block, scale):
        return tuple(t.new_empty(t.shape) for t in (q, k, v))

    @fake("speed3r_b200::sel_attn_bwd_pooled")
    def _(q, k, v, idx, lse, delta, do_s, dq_c, dk_c, dv_c, block, kernel, stride, scale):
        return tuple(t.new_empty(t.shape) for t in (q, k, v))

    @fake("speed3r_b200::pool_qkv_fwd")
    def _(q, k, v, block, kernel, stride):
        window = lambda x, kernel, stride: x.new_empty(*x.shape[:2], (x.shape[2] - kernel) // stride + 1, x.shape[3])
        return window(q, block, block), window(k, kernel, stride), window(v, kernel, stride)

    @fake("speed3r_b200::prologue_fwd")
    def _(qkv, heads, block, pos, cos, sin, qw, qb, kw, kb, eps):
        B, N = qkv.shape[:2]
        d = qkv.numel() // (B * N * 3 * heads)
        return tuple(qkv.new_empty(B, heads, n, d) for n in (N, N, N, N // block, N // block, N // block))

    @fake("speed3r_b200::prologue_bwd")
    def _(qkv, heads, block, pos, cos, sin, qw, kw, eps, dq, dk, dv, dq_c, dk_c, dv_c):
        return (qkv.new_empty(qkv.shape),
                qkv.new_empty((0,) if qw is None else (4, dq.shape[-1]), dtype=torch.float32))

    @fake("speed3r_b200::delta")
    def _(o, d_o):
        return o.new_empty(o.shape[:-1], dtype=torch.float32)

    @fake("speed3r_b200::merge_bwd")
    def _(dy, gate, o_c, o_s, block):
        B, H, Tq, d = o_s.shape
        return (o_s.new_empty(o_s.shape), o_s.new_empty(B, H, Tq, 2, dtype=torch.float32), o_c.new_empty(o_c.shape),
                o_s.new_empty(B, H, Tq, dtype=torch.float32))

    @fake("speed3r_b200::residual_norm_fwd")
    def _(x, y, weight, bias, scale, gate, post_weight, post_bias, norm, post, kind, eps, post_eps, h_type, keep):
        return (x.new_empty(x.shape if y is not None else (0,)), x.new_empty(x.shape if norm else (0,), dtype=h_type),
                x.new_empty(4 if keep else 0, x.shape[0] * x.shape[1], dtype=torch.float32))

    @fake("speed3r_b200::residual_norm_bwd")
    def _(r, y, weight, scale, gate, post_weight, post_bias, stats, dr, dh, branch, post, kind, want, param_type):
        if dh is None:
            want &= ~12
        of = lambda bit: r.new_empty(r.shape[2] if want & bit else 0, dtype=param_type)
        return [r.new_empty(r.shape), r.new_empty(r.shape, dtype=branch) if want & 2 and branch is not None else r.new_empty(0), of(4), of(8), of(16),
                gate.new_empty(gate.shape) if want & 32 else r.new_empty(0), of(64), of(128)]

    @fake("speed3r_b200::residual_norm_int8")
    def _(x, y, weight, bias, scale, gate, post_weight, post_bias, post, kind, eps, post_eps):
        B, T, C = x.shape
        return (x.new_empty(x.shape if y is not None else (0,)), x.new_empty(B, T, -(-C // 16) * 16, dtype=torch.int8).narrow(2, 0, C),
                x.new_empty(B, T, dtype=torch.float32))

    @fake("speed3r_b200::quantize_rows")
    def _(x):
        K = x.shape[-1]
        return (x.new_empty(x.numel() // K, -(-K // 16) * 16, dtype=torch.int8).narrow(1, 0, K).view(x.shape),
                x.new_empty(x.shape[:-1], dtype=torch.float32))

    @fake("speed3r_b200::int8_product")
    def _(q, q_scale, weight, weight_scale, bias, out_type):
        return q.new_empty(*q.shape[:-1], weight.shape[0], dtype=out_type)

    @fake("speed3r_b200::norm_of")
    def _(tensors):
        return tensors[0].new_empty((), dtype=torch.float32)

    fake("speed3r_b200::adamw_update", lambda *a: None)
    fake("speed3r_b200::adamw_values", lambda *a: None)


def _ops():
    """The ``torch.ops`` namespace of the native operators, loaded (and built if need be) at first use."""
    global _ns
    if _ns is None:
        with _lock:
            if _ns is None:
                _lib.load()
                torch.ops.load_library(_lib.TORCH_LIB_PATH)
                _register_fakes()
                _ns = torch.ops.speed3r_b200
    return _ns


def _need(t: Tensor, name: str, dtype=_BF16, contiguous=True) -> None:
    if not t.is_cuda:
        raise RuntimeError(f"{name} must be a CUDA tensor: the speed3r_b200 kernels have no CPU path")
    if t.dtype != dtype:
        raise RuntimeError(f"{name} must be {dtype}, got {t.dtype}")
    if contiguous and not t.is_contiguous():
        raise RuntimeError(f"{name} must be contiguous")


def _scale(softmax_scale: Optional[float], q: Tensor) -> float:
    return 1.0 / math.sqrt(q.shape[-1]) if softmax_scale is None else float(softmax_scale)


# ------------------------------------------------------------------------------------------------
# raw kernels (no autograd)
# ------------------------------------------------------------------------------------------------
def _cmp_fwd(q_c: Tensor, k_c: Tensor, v_c: Tensor, topk: int, scale: float) -> Tuple[Tensor, Tensor, Tensor]:
    """(o, lse, idx) of the compression attention."""
    return _ops().cmp_attn_topk_fwd.default(q_c, k_c, v_c, topk, scale)


def _sel_fwd(q: Tensor, k: Tensor, v: Tensor, idx: Tensor, gate: Optional[Tensor], o_c: Optional[Tensor],
             block: int, scale: float, want_o: bool, want_lse: bool, kv_chunks: int) -> Tuple[Tensor, Tensor, Tensor]:
    """Returns (o_s, lse_s, y); tensors not asked for come back with zero elements."""
    return _ops().sel_attn_fwd.default(q, k, v, idx, gate, o_c, block, scale, want_o, want_lse, kv_chunks)


def build_key_csr(idx: Tensor, num_key_blocks: int) -> Tuple[Tensor, Tensor]:
    """Key-centric CSR of the selection table: (offsets [B,H,Nkb+1], qids [B,H,Nq*K]) int32."""
    return _ops().build_key_csr.default(idx, num_key_blocks)


def qkv_prologue(qkv: Tensor, num_heads: int, block: int, pos: Optional[Tensor] = None,
                 cos: Optional[Tensor] = None, sin: Optional[Tensor] = None,
                 q_norm: Optional[Tuple[Tensor, Tensor, float]] = None,
                 k_norm: Optional[Tuple[Tensor, Tensor, float]] = None):
    """Everything between the qkv projection and the two attention calls of the module
    (pi3/models/layers/sparse_attention.py:95-123) in one kernel, forward only:
    ``qkv [B,N,3*H*d]`` -> ``(q, k, v [B,H,N,d], q_c, k_c, v_c [B,H,N/block,d])`` with the per-head
    LayerNorm of q and k (``(weight, bias, eps)`` or None), the 2-D rotary embedding at ``pos
    [B,N,2]`` (``cos``/``sin`` = the bf16 tables RoPE2D caches) and, for the pooled tensors, at each
    block's truncated mean position."""
    _need(qkv, "qkv")
    if qkv.requires_grad and torch.is_grad_enabled():
        raise RuntimeError("qkv_prologue is forward-only; the module's training path uses its differentiable form")
    with torch.no_grad():
        return _prologue(qkv, num_heads, block, pos, cos, sin, q_norm, k_norm)


def _prologue(qkv, num_heads, block, pos, cos, sin, q_norm, k_norm):
    """``qkv_prologue`` with a backward."""
    if (q_norm is None) != (k_norm is None):
        raise RuntimeError("qkv_prologue: q_norm and k_norm come together or not at all")
    if q_norm is not None and abs(q_norm[2] - k_norm[2]) > 0:
        raise RuntimeError("qkv_prologue: q_norm and k_norm must share eps")
    qw, qb, eps = q_norm if q_norm is not None else (None, None, 1e-5)
    kw, kb, _ = k_norm if k_norm is not None else (None, None, 0.0)
    return _ops().prologue.default(qkv, num_heads, block, pos, cos, sin, qw, qb, kw, kb, float(eps))


# ------------------------------------------------------------------------------------------------
# differentiable operators
# ------------------------------------------------------------------------------------------------
def pool_tokens(x: Tensor, kernel: int = 16, stride: int = 16) -> Tensor:
    """Mean over ``kernel`` consecutive tokens every ``stride`` tokens of ``x [B,H,T,d]`` (any
    batch/head/token strides) -> ``[B,H,Nc,d]``.  sparse_attention.py:97-102 for one of q/k/v."""
    return _ops().pool_tokens.default(x, kernel, stride)


def flash_attn_blocktopk_func(q, k, v, topk_val, group, take, softmax_scale=None):
    """Compression attention whose table ranks selection BLOCKS by the softmax mass of their own compressed
    keys (columns ``group*n .. group*n+take-1``): for settings where compressed keys are finer than selection
    blocks.  Returns ``(o, idx)`` like ``flash_attn_topk_func``; ``idx`` holds block numbers."""
    if int(group) < 1:
        raise RuntimeError(f"flash_attn_blocktopk_func: {group} compressed keys per block")
    return _ops().flash_attn_topk.default(q, k, v, int(topk_val), _scale(softmax_scale, q), int(group), int(take))


def sparse_attention_op(q, k, v, gate, block_size=16, topk=32, kernel=16, stride=16):
    """The whole op on ``q,k,v [B,H,T,d]`` and ``gate [B,H,T,2]``: queries pooled per selection block
    (``block_size`` tokens), keys and values pooled with ``kernel``/``stride``, compression attention with the
    fused table, selection attention over the table's blocks, gated merge.  At 16/16/16 this is the
    reference's path (``sparse_attention.py:95-136`` without the norms and rotary embedding); when compressed
    keys are finer than selection blocks (e.g. kernel 32, stride 16, blocks of 64) the blocks are ranked by
    probability mass.  Returns ``(y [B,T,H*d], idx)``."""
    group = take = 0
    if (kernel, stride) != (block_size, block_size):
        if block_size % stride or kernel > block_size or (block_size - kernel) % stride:
            raise RuntimeError("need stride | block_size and kernel = block_size - i*stride")
        group, take = block_size // stride, (block_size - kernel) // stride + 1
    return _ops().sparse_attention.default(q, k, v, gate, int(block_size), int(topk), int(kernel), int(stride),
                                           _scale(None, q), group, take)


def flash_attn_topk_func(q, k, v, topk_val, bias=None, causal=False, softmax_scale=None):
    """Compression attention with fused top-k selection; drop-in for the reference's
    ``flash_attn_topk_func`` (flash_attention_topk.py:633-668).  Inputs ``[B,H,n,d]`` bf16."""
    assert bias is None, "bias is not supported (the reference ignores it as well)"
    assert not causal, "the sparse global attention is bidirectional; causal is not implemented"
    return _ops().flash_attn_topk.default(q, k, v, int(topk_val), _scale(softmax_scale, q), 0, 0)


def topk_blocksparse_attention(q, k, v, topk_idx, block_size, softmax_scale=None):
    """Block-sparse selection attention; drop-in for the reference's ``topk_blocksparse_attention``
    (topk_blocksparse_attention.py:1093-1121).  q,k,v ``[B,H,T,d]`` bf16 contiguous, ``topk_idx``
    ``[B,H,T/block,K]`` int32."""
    assert q.dtype == torch.bfloat16, "bf16 only"
    assert q.dtype == k.dtype and k.dtype == v.dtype
    assert topk_idx.dtype == torch.int32
    return _ops().topk_blocksparse.default(q, k, v, topk_idx, int(block_size), _scale(softmax_scale, q))


def sel_attn_merge(q, k, v, topk_idx, gate, o_c, block_size, softmax_scale=None):
    """Selection attention with the gated merge fused into its epilogue:
    ``y[b,t,(h d)] = gate[b,h,t,0] * o_c[b,h,t//block] + gate[b,h,t,1] * sel_attn(q,k,v)[b,h,t]``
    (topk_blocksparse_attention.py:35-128 + sparse_attention.py:127-136).  ``gate [B,H,T,2]`` may
    be a strided view of the ``[B,T,2H]`` projection."""
    return _ops().sel_merge.default(q, k, v, topk_idx, gate, o_c, int(block_size), _scale(softmax_scale, q))


def sel_attn_merge_chunked(q, k_chunks, v_chunks, topk_idx, gate, o_c, block_size, softmax_scale=None):
    """Forward-only form of ``sel_attn_merge`` for sequence-partitioned inference: the keys and
    values are the all-gathered ``[G,B,H,Tk/G,d]`` chunks (rank order = sequence order), read in
    place; ``q``, ``gate``, ``o_c`` and ``topk_idx`` are the local query rows; ``topk_idx`` holds
    GLOBAL key-block numbers."""
    with torch.no_grad():
        return _sel_fwd(q, k_chunks, v_chunks, topk_idx, gate, o_c, int(block_size), _scale(softmax_scale, q),
                        False, False, int(k_chunks.shape[0]))[2]


# ------------------------------------------------------------------------------------------------
# the rest of a block: residual, LayerScale, gate and norms; 8-bit products; the optimiser's step
# ------------------------------------------------------------------------------------------------
_KINDS = {"layer": 0, "rms": 1}
NORM_TYPES = (torch.float32, torch.bfloat16, torch.float16)
NORM_MAX_CHANNELS = 8192


def _norm_args(norm, post_norm, kind):
    if kind not in _KINDS:
        raise RuntimeError(f"residual_norm: kind must be 'layer' or 'rms', got {kind!r}")
    w, b, eps = norm if norm is not None else (None, None, 0.0)
    pw, pb, post_eps = post_norm if post_norm is not None else (None, None, 0.0)
    return w, b, float(eps), pw, pb, float(post_eps)


def residual_norm(x: Tensor, y: Optional[Tensor] = None, norm=None, scale: Optional[Tensor] = None, gate: Optional[Tensor] = None,
                  post_norm=None, kind: str = "layer", out_dtype: Optional[torch.dtype] = None):
    """What stands between two sub-layers of a block (pi3/models/layers/block.py:310-335, LayerScale and residual, then the
    next norm), in one pass and with gradients::

        u = y, or post_norm(y)
        r = x + u * scale * gate            (in x's type)
        h = norm(r)                         (in ``out_dtype``, by default x's type)

    ``x``, ``y`` ``[.., T, C]`` fp32, bf16 or fp16, each of its own type, C up to 8192.  ``norm`` and ``post_norm`` are
    ``(weight, bias, eps)``, weight and bias ``[C]`` or None; ``kind`` says whether they are LayerNorms (``"layer"``) or divide by
    the root of the mean square (``"rms"``).  ``scale [C]`` is the LayerScale, ``gate`` a factor per token ``[.., T, 1]``, per
    sample ``[.., 1, 1]`` (stochastic depth) or per sample and channel ``[.., 1, C]`` (modulation).  Returns ``(r, h)``: ``r`` is
    ``x`` itself where ``y`` is None, ``h`` is None where ``norm`` is None.  The norm is that of ``r`` as it is stored."""
    w, b, eps, pw, pb, post_eps = _norm_args(norm, post_norm, kind)
    h_type = x.dtype if out_dtype is None else out_dtype
    if h_type not in NORM_TYPES:
        raise RuntimeError(f"residual_norm: out_dtype must be fp32, bf16 or fp16, got {h_type}")
    r, h = _ops().residual_norm.default(x, y, w, b, scale, gate, pw, pb, norm is not None, post_norm is not None, _KINDS[kind], eps,
                                        post_eps, h_type)
    return r if y is not None else x, h if norm is not None else None


def residual_norm_int8(x: Tensor, y: Optional[Tensor] = None, norm=None, scale: Optional[Tensor] = None,
                       gate: Optional[Tensor] = None, post_norm=None, kind: str = "layer"):
    """``residual_norm`` without gradients whose ``h`` leaves as 8-bit tokens: ``(r, q, q_scale)`` as ``quantize_tokens`` makes
    them of ``h``, without ``h`` being written."""
    if norm is None:
        raise RuntimeError("residual_norm_int8 needs a norm")
    w, b, eps, pw, pb, post_eps = _norm_args(norm, post_norm, kind)
    r, q, s = _ops().residual_norm_to_int8.default(x, y, w, b, scale, gate, pw, pb, post_norm is not None, _KINDS[kind], eps, post_eps)
    return x if y is None else r, q, s


def quantize_tokens(x: Tensor) -> Tuple[Tensor, Tensor]:
    """``x [.., K]`` fp32, bf16 or fp16 as 8-bit integers with a scale per token: ``q = round(x / q_scale)`` with
    ``q_scale [..] = max|x| / 127``.  Rows of ``q`` lie a multiple of 16 bytes apart.  The rows of a weight ``[N, K]`` become
    its output channels.  No gradients."""
    if x.requires_grad and torch.is_grad_enabled():
        raise RuntimeError("quantize_tokens is forward-only: call it under torch.no_grad()")
    return _ops().quantize_tokens.default(x)


def int8_linear(q: Tensor, q_scale: Tensor, weight: Tensor, weight_scale: Tensor, bias: Optional[Tensor] = None,
                out_dtype: torch.dtype = _BF16) -> Tensor:
    """``(q @ weight.T) * q_scale * weight_scale + bias`` for ``q [.., K]`` and ``weight [N, K]`` of 8-bit integers: exact sums in
    32 bits, one fp32 scale per token and per output channel, fp32 ``bias [N]``, one rounding to ``out_dtype``.  No gradients."""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q_scale, weight_scale, bias)):
        raise RuntimeError("int8_linear is forward-only: call it under torch.no_grad()")
    if out_dtype not in NORM_TYPES:
        raise RuntimeError(f"int8_linear: out_dtype must be fp32, bf16 or fp16, got {out_dtype}")
    return _ops().int8_linear.default(q, q_scale, weight, weight_scale, bias, out_dtype)


@torch.no_grad()
def grad_norm(tensors) -> Tensor:
    """Euclidean norm of all elements of a list of tensors (one device; fp32, bf16, fp16), as a 0-dim fp32 tensor: squares summed
    in 64 bits in a fixed order, without a synchronisation."""
    return _ops().grad_norm.default(list(tensors))


@torch.no_grad()
def adamw_step(params, grads, exp_avg, exp_avg_sq, step: Tensor, lr=1e-3, betas=(0.9, 0.999), eps: float = 1e-8,
               weight_decay: float = 1e-2, grad_norm: Optional[Tensor] = None, max_norm: Optional[float] = None, scales=None,
               seed: Optional[int] = None, numbers=None) -> None:
    """One AdamW step in place over lists of tensors of one device, in one pass::

        g = grad * min(1, max_norm / (grad_norm + 1e-6))         (with max_norm)
        m = beta1 m + (1 - beta1) g;   v = beta2 v + (1 - beta2) g^2
        p = p (1 - lr weight_decay) - lr / (1 - beta1^t) * m / (sqrt(v / (1 - beta2^t)) + eps)

    ``step`` is a 0-dim int64 tensor on the device that becomes t; ``lr`` a number or a 0-dim fp32 tensor on the device.  ``eps`` is
    0 or at least 2^-126.  Where ``grad_norm`` is given and not finite, nothing changes.  States are fp32, or, where ``scales`` (a list, entries may be None) has a
    uint8 ``[2, ceil(n / 256)]`` for a tensor, uint8 codes: see ``adamw_state``.  With ``seed`` (0 to 2^63 - 1) what is kept in fewer
    bits than 32 - 8-bit states, bf16 parameters - is rounded stochastically, the same way for the same seed and step; without it to
    nearest.  A tensor's random numbers go by its index in the lists, or by its entry in ``numbers`` (one integer below 2^24 per
    tensor): give every tensor its own where several calls make up a step.  Parameters: fp32, bf16 or fp16, contiguous."""
    if seed is not None and not 0 <= int(seed) < 1 << 63:
        raise RuntimeError(f"adamw_step: seed {seed}")
    if max_norm is not None and not max_norm > 0:
        raise RuntimeError(f"adamw_step: max_norm {max_norm}")
    if max_norm is not None and grad_norm is None:
        raise RuntimeError("adamw_step: max_norm needs grad_norm")
    on_device = isinstance(lr, Tensor)
    _ops().adamw_step.default(list(params), list(grads), list(exp_avg), list(exp_avg_sq), step, [] if scales is None else list(scales),
                              0.0 if on_device else float(lr), lr if on_device else None, float(betas[0]), float(betas[1]), float(eps),
                              float(weight_decay), grad_norm, 0.0 if max_norm is None else float(max_norm), -1 if seed is None else int(seed),
                              None if numbers is None else list(numbers))


@torch.no_grad()
def adamw_state(exp_avg, exp_avg_sq, scales, out=None):
    """``(m, v)``, two lists of fp32 tensors: what 8-bit states stand for.  Blocks of 256 codes share a power of two; a code of ``m``
    has a sign, 4 bits of exponent and 3 of mantissa, one of ``v`` 5 and 3.  ``out``: two lists to write into."""
    m, v = out if out is not None else tuple([torch.empty(t.shape, dtype=torch.float32, device=t.device) for t in exp_avg] for _ in range(2))
    _ops().adamw_state.default(list(exp_avg), list(exp_avg_sq), list(scales), list(m), list(v))
    return m, v
