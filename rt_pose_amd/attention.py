"""Cross attention to an encoder's states of another length, on csrc/cross_attn.hip.

    cross_attention(q, k, v, key_lens=None, key_mask=None, scale=None)      [batch, queries, heads, dim]

q: [b, sq, hq, d]; k, v: [b, sk, hkv, d] with hq a multiple of hkv (head h reads k and v of head h // (hq // hkv)).  Of batch entry i the keys j
with j < key_lens[i] and key_mask[i, j] count.  Keys that do not count -- an encoder's padding -- are never multiplied, whatever they hold (NaN
too), and get zero gradients; a row without keys gives zeros, and so does one whose every score is minus infinity.  bf16 or fp16, d a multiple of 8 up to 128; any strides (a tensor whose rows
are not 16-byte aligned is copied).  Scores, softmax statistics and sums are fp32.  For the second products (with v; with k, q and o's gradient) the
exponentials and the scores' gradients are rounded once to the operands' type with more than 32 query rows of a key head (sq * hq / hkv); with up to
32 both halves of them are kept.  The result does not depend on scheduling.  Differentiable in q, k and v
(backward; a forward-mode tangent is refused with NotImplementedError).  A trace holds the operator as one node, which checks its arguments at every call.
With few queries (single tokens while serving, key-point queries) the keys are split over the GPU and joined.
Errors as in rt_pose_amd.rmsnorm.
"""
import ctypes as C

import torch

from . import _lib
from ._tokens import DTYPES, TokenFunction, call, like, once, p, same_device


def _check(q, k, v, key_lens, key_mask, scale):
    same_device(q, k, v, key_lens, key_mask)
    dtype, qs, ks = q.dtype, q.shape, k.shape
    if dtype != torch.bfloat16 and dtype != torch.float16:
        raise NotImplementedError("cross_attention: bf16 or fp16 only (got %s)" % dtype)
    if k.dtype != dtype or v.dtype != dtype:
        raise ValueError("cross_attention: q, k and v of one type expected (got %s, %s, %s)" % (dtype, k.dtype, v.dtype))
    if len(qs) != 4 or len(ks) != 4 or ks != v.shape or qs[0] != ks[0] or qs[3] != ks[3]:
        raise ValueError("cross_attention: [b, sq, hq, d] and twice [b, sk, hkv, d] expected (got %s, %s, %s)" % (tuple(qs), tuple(ks), tuple(v.shape)))
    if ks[2] < 1 or qs[2] < 1 or qs[2] % ks[2]:
        raise ValueError("cross_attention: %d query heads are no multiple of %d key heads" % (qs[2], ks[2]))
    if qs[3] < 8 or qs[3] % 8 or qs[3] > 128:
        raise NotImplementedError("cross_attention: head widths of a multiple of 8 up to 128 (got %d)" % qs[3])
    if key_lens is not None and (key_lens.shape != qs[:1] or key_lens.dtype not in (torch.int32, torch.int64)):
        raise ValueError("cross_attention: key_lens of shape (%d,) and whole numbers expected (got %s %s)" % (qs[0], tuple(key_lens.shape), key_lens.dtype))
    if key_mask is not None and key_mask.dtype != torch.bool:
        raise NotImplementedError("cross_attention: key_mask of truth values only, True where a key counts (got %s)" % key_mask.dtype)
    if key_mask is not None and key_mask.shape != ks[:2]:
        raise ValueError("cross_attention: key_mask of shape %s expected (got %s)" % (tuple(ks[:2]), tuple(key_mask.shape)))
    if max(qs[0], qs[1], qs[2], ks[1]) > 1 << 30:
        raise ValueError("cross_attention: sizes beyond 2^30 (got %s and %s)" % (tuple(qs), tuple(ks)))
    if not 1e-45 < scale <= 2e38:
        raise ValueError("cross_attention: a positive, finite scale expected (got %r)" % (scale,))


def _aligned(t, group=0):
    """t with contiguous heads in rows on 16-byte boundaries: itself, or a copy.  The kernels index 64 tokens, and `group` heads, in 32 bits."""
    if t.data_ptr() % 16 == 0:
        if t.is_contiguous():
            return t
        st = t.stride()
        if st[3] == 1 and st[1] <= 1 << 23 and st[2] * group <= 1 << 28 and all(s % 8 == 0 or n == 1 for s, n in zip(st, t.shape[:3])):
            return t
    return t.contiguous() if not t.is_contiguous() else t.clone()


def _strides(t):
    """of batch, token and head; of a dimension of one any would do, and a tensor may have any there"""
    if t.is_contiguous():
        _, n, h, d = t.shape
        return n * h * d, h * d, d
    return tuple(s if n > 1 else 0 for s, n in zip(t.stride()[:3], t.shape))


def _operands(q, k, v, key_lens, key_mask, scale):
    b, sq, hq, d = q.shape
    _, sk, hkv, _ = k.shape
    return _lib.RtpXattn(q.data_ptr(), k.data_ptr(), v.data_ptr(), *_strides(q), *_strides(k), *_strides(v), p(key_mask),
                         *((0, 0) if key_mask is None else key_mask.stride()), p(key_lens), b, sq, sk, hq, hkv, d, DTYPES[q.dtype], scale)


def _workspace(a, backward, ref):
    n = _lib.load().rtp_xattn_workspace_bytes(C.byref(a), backward)
    if n < 0:
        raise _lib.RtpError("cross_attention: sizes beyond what the kernels index (%s)" % (tuple(ref.shape),))
    return ref.new_empty(n, dtype=torch.uint8) if n else None, n


def _forward(a, q, o_lo=None, lse=None):
    o = like(q)
    if o.numel():
        ws, n = _workspace(a, 0, q)
        call("rtp_xattn_forward", q, C.byref(a), p(o), p(o_lo), p(lse), p(ws), n)
    return o


class CrossAttentionFunction(TokenFunction):
    @staticmethod
    def forward(ctx, q, k, v, key_lens, key_mask, scale, keep):
        """keep: whether a backward pass may follow, if an input asks for its gradient."""
        scale = float(q.shape[-1]) ** -0.5 if scale is None and q.dim() == 4 and q.shape[-1] else 1.0 if scale is None else float(scale)
        _check(q, k, v, key_lens, key_mask, scale)
        q, k, v = _aligned(q, q.shape[2] // k.shape[2]), _aligned(k), _aligned(v)
        if key_lens is not None:
            key_lens = (key_lens if key_lens.dtype == torch.int32 else key_lens.clamp(0, k.shape[1]).to(torch.int32)).contiguous()
        a = _operands(q, k, v, key_lens, key_mask, scale)
        need = ctx.needs_input_grad
        if not (keep and (need[0] or need[1] or need[2])):
            return _forward(a, q)
        n = q.shape[:3].numel()
        if key_mask is not None:                    # room for its bits behind
            n = -(-n // 64) * 64 + q.shape[0] * 4 * -(-k.shape[1] // 128)
        o_lo, lse = like(q), q.new_empty(n, dtype=torch.float32)
        o = _forward(a, q, o_lo, lse)
        ctx.operands, ctx.scale, ctx.layout = a, scale, (q.stride(), k.stride(), v.stride())
        ctx.save_for_backward(q, k, v, key_lens, key_mask, o, o_lo, lse)
        return o

    @staticmethod
    @once
    def backward(ctx, do):
        q, k, v, key_lens, key_mask, o, o_lo, lse = ctx.saved_tensors
        need_q, need_k, need_v = ctx.needs_input_grad[:3]
        dq = like(q) if need_q else None
        dk, dv = (like(k), like(v)) if need_k or need_v else (None, None)
        if q.numel() == 0 or k.numel() == 0:
            return tuple(None if t is None else t.zero_() for t in (dq, dk, dv)) + (None,) * 4
        a, do = ctx.operands, _aligned(do, q.shape[2] // k.shape[2])
        if a.q != q.data_ptr() or a.k != k.data_ptr() or a.v != v.data_ptr() or a.key_lens != p(key_lens) or a.key_mask != p(key_mask) or ctx.layout != (
                q.stride(), k.stride(), v.stride()):
            q, k, v = _aligned(q, q.shape[2] // k.shape[2]), _aligned(k), _aligned(v)          # saved tensors were kept elsewhere meanwhile
            a = _operands(q, k, v, key_lens, key_mask, ctx.scale)
        ws, n = _workspace(a, 1, q)
        call("rtp_xattn_backward", q, C.byref(a), p(o), p(o_lo), p(lse), p(do), *_strides(do), p(dq), p(dk), p(dv), p(ws), n)
        return dq, dk, dv, None, None, None, None


def cross_attention(q, k, v, key_lens=None, key_mask=None, scale=None):
    """scale: 1 / sqrt(d) by default.  key_lens: [b] int32 or int64 (taken between 0 and sk); key_mask: [b, sk], True where a key counts."""
    return CrossAttentionFunction.apply(q, k, v, key_lens, key_mask, scale, torch.is_grad_enabled() or torch.jit.is_tracing())
