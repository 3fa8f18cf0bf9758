"""Root-mean-square norm of token rows with the residual's addition, on the HIP kernels of csrc/token_norm.hip.

    rms_norm(x, weight, eps)                       y
    add_rms_norm(x, residual, weight, eps)         y, stream      stream = x + residual in x's type, y = stream / rms(stream) * weight
    add_rms_norm_fp8(x, residual, weight, eps)     q, scale, stream      y in 8 bits, one scale for 128 columns (rt_pose_amd.fp8)
    RMSNorm(dim)                                   module over the first two

x, residual: [..., dim] of one type (fp32, fp16, bf16), any strides; weight: [dim], of that type or fp32.  Differentiable in x, residual
and weight (not in the 8-bit form; forward-mode tangents are refused with NotImplementedError); the sums are fp32 and the gradients do not
depend on scheduling.  A trace holds each call as one node, which checks its arguments every time.  Error behaviour as in
rt_pose_amd.dcn: CPU tensors -> NotImplementedError, a wrong type -> NotImplementedError, shapes that do not fit -> ValueError,
a failing native call -> RtpError.
"""
import torch
import torch.nn as nn

from . import _lib
from ._tokens import DTYPES, TokenFunction, call, fp8_rows, like, once, p, rows_of, same_device, without_gradient


def _check(x, residual, weight):
    same_device(x, residual, weight)
    if x.dtype not in DTYPES:
        raise NotImplementedError("rms norm: fp32, fp16 or bf16 rows only (got %s)" % x.dtype)
    shape = x.shape
    if len(shape) < 1 or shape[-1] < 1:
        raise ValueError("rms norm: rows of at least one column expected (got shape %s)" % (tuple(shape),))
    if shape[-1] > 16384:
        raise NotImplementedError("rms norm: rows of up to 16384 columns (got %d)" % shape[-1])
    if residual is not None and (residual.shape != shape or residual.dtype != x.dtype):
        raise ValueError("rms norm: the residual must have x's shape and type (got %s %s beside %s %s)"
                         % (tuple(residual.shape), residual.dtype, tuple(x.shape), x.dtype))
    if weight.shape != shape[-1:]:
        raise ValueError("rms norm: weight of shape (%d,) expected (got %s)" % (x.shape[-1], tuple(weight.shape)))
    if weight.dtype != x.dtype and weight.dtype != torch.float32:
        raise NotImplementedError("rms norm: weight in x's type or fp32 (got %s beside %s)" % (weight.dtype, x.dtype))


def _forward(x, residual, weight, eps):
    x2, w = rows_of(x), weight.contiguous()
    r2 = rows_of(residual) if residual is not None else None
    y = like(x)
    s = torch.empty_like(y) if residual is not None else None
    call("rtp_rmsnorm_forward", x, p(x2), x2.stride(0), p(r2), 0 if r2 is None else r2.stride(0), p(w), DTYPES[w.dtype], p(y), p(s), *x2.shape,
         DTYPES[x.dtype], eps)
    return y, s


def _backward(s, weight, eps, dy, ds, need_w):
    """dx (also the residual's gradient) and, if need_w, dw of the rows `s` that were normed."""
    s2, w = rows_of(s), weight.contiguous()
    rows, h = s2.shape
    dx, dw = like(s), torch.empty_like(w) if need_w else None
    if rows == 0:
        return dx, dw.zero_() if need_w else None
    dy2, ds2 = rows_of(dy), rows_of(ds) if ds is not None else None
    part = s.new_empty(_lib.load().rtp_rmsnorm_backward_slots(rows, h) * h, dtype=torch.float32) if need_w else None
    call("rtp_rmsnorm_backward", s, p(s2), s2.stride(0), p(w), DTYPES[w.dtype], p(dy2), dy2.stride(0), p(ds2), 0 if ds2 is None else ds2.stride(0),
         p(dx), p(dw), p(part), rows, h, DTYPES[s.dtype], eps)
    return dx, dw


class RMSNormFunction(TokenFunction):
    @staticmethod
    def forward(ctx, x, weight, eps):
        _check(x, None, weight)
        ctx.eps = eps
        ctx.save_for_backward(x, weight)
        return _forward(x, None, weight, eps)[0]

    @staticmethod
    @once
    def backward(ctx, dy):
        x, weight = ctx.saved_tensors
        dx, dw = _backward(x, weight, ctx.eps, dy, None, ctx.needs_input_grad[1])
        return dx, dw, None


class AddRMSNormFunction(TokenFunction):
    @staticmethod
    def forward(ctx, x, residual, weight, eps):
        _check(x, residual, weight)
        y, s = _forward(x, residual, weight, eps)
        ctx.eps = eps
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(s, weight)
        return y, s

    @staticmethod
    @once
    def backward(ctx, dy, ds):
        s, weight = ctx.saved_tensors
        if dy is None:                  # only the stream was used
            return ds, ds, None, None
        dx, dw = _backward(s, weight, ctx.eps, dy, ds, ctx.needs_input_grad[2])
        return dx, dx, dw, None


class AddRMSNormFp8Function(TokenFunction):
    @staticmethod
    def forward(ctx, x, residual, weight, eps):
        _check(x, residual, weight)
        x2, w = rows_of(x), weight.contiguous()
        r2 = rows_of(residual) if residual is not None else None
        q, scale = fp8_rows(x.shape, x.device)
        s = torch.empty(x.shape, dtype=x.dtype, device=x.device) if residual is not None else None
        call("rtp_rmsnorm_fp8_forward", x, p(x2), x2.stride(0), p(r2), 0 if r2 is None else r2.stride(0), p(w), DTYPES[w.dtype], p(q),
             -(-x.shape[-1] // 16) * 16, p(scale), p(s), *x2.shape, DTYPES[x.dtype], float(eps))
        return without_gradient(ctx, q, scale) if s is None else without_gradient(ctx, q, scale, s)


def rms_norm(x, weight, eps=1e-6):
    return RMSNormFunction.apply(x, weight, float(eps))


def add_rms_norm(x, residual, weight, eps=1e-6):
    if residual is None:
        raise ValueError("add_rms_norm: a residual is expected (rms_norm has none)")
    return AddRMSNormFunction.apply(x, residual, weight, float(eps))


def add_rms_norm_fp8(x, residual, weight, eps=1e-6):
    """For serving: the normed rows in 8 bits and their scales, as rt_pose_amd.fp8.matmul_fp8 reads them, and the stream.  residual may be
    None (the stream is x itself).  The value that is quantised is the fp32 one.  Not differentiable: the outputs carry no gradient, a
    forward-mode tangent is refused with NotImplementedError."""
    out = AddRMSNormFp8Function.apply(x, residual, weight, float(eps))
    return out if residual is not None else (*out, x)


class RMSNorm(nn.Module):
    """y = rms_norm(x); with a residual (y, stream) = add_rms_norm(x, residual)."""

    def __init__(self, dim, eps=1e-6):
        super().__init__()
        self.dim, self.eps = dim, eps
        self.weight = nn.Parameter(torch.ones(dim))

    def forward(self, x, residual=None):
        return rms_norm(x, self.weight, self.eps) if residual is None else add_rms_norm(x, residual, self.weight, self.eps)

    def extra_repr(self):
        return "%d, eps=%g" % (self.dim, self.eps)
