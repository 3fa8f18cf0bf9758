"""Marshalling shared by the token operators (rmsnorm.py, fp8.py, attention.py).  Small calls are bound by the host: one native call, no
context manager and no stream object where the tensor's device is already the current one."""
import torch
from torch.autograd import Function, forward_ad
from torch.autograd.function import once_differentiable

from . import _lib

DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}   # RTP_DT_* of include/rtp.h
FP8 = torch.float8_e4m3fn


def p(t):
    return None if t is None else t.data_ptr()


# the current stream's handle without a Stream object around it: 0.1 us instead of 1.2, and 15 us less in a backward pass, whose thread is another
_raw_stream, _current_device = torch._C._cuda_getCurrentRawStream, torch._C._cuda_getDevice


def _recorded_by_fx():
    from torch.fx.experimental.proxy_tensor import get_proxy_mode
    return get_proxy_mode() is not None


def call(name, t, *args):
    """The native entry `name` on the current stream of t's device, with that device current; RtpError if it fails.  Refused under make_fx, which sees
    torch's operators alone: its graph would hold the output's allocation and not the call."""
    if torch._C._len_torch_dispatch_stack() and _recorded_by_fx():
        raise NotImplementedError("rt_pose_amd: the token operators cannot be recorded by make_fx")
    index = t.get_device()
    if index == _current_device():
        rc = getattr(_lib.load(), name)(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = getattr(_lib.load(), name)(*args, _raw_stream(index))
    if rc != 0:
        _lib.check(rc, name)


class TokenFunction(Function):
    """What every token operator's call goes through, where nothing asks for a gradient too: only a Function's call is seen by forward mode, whose
    tangents would be dropped without a word, and by a trace, which would hold the output's allocation and not the operator.  Arguments are checked and
    laid out inside `forward`: a trace repeats that, and nothing else, with the tensors of its later calls."""

    @staticmethod
    def jvp(ctx, *tangents):
        raise NotImplementedError("rt_pose_amd: the token operators have no forward-mode derivatives")


def without_gradient(ctx, *outputs):
    """A Function's outputs that carry no gradient, whatever the inputs ask for."""
    if True in ctx.needs_input_grad:
        ctx.mark_non_differentiable(*outputs)
    return outputs


def once(backward):
    """A Function's backward that cannot be differentiated again: autograd says so if one tries, and tangents of the outputs' gradients are refused like
    the inputs'.  The guard is put on only where a graph of the
    backward pass is asked for: a backward pass runs in a thread of its own, where every line of Python costs twice."""
    guarded = once_differentiable(backward)

    def run(ctx, *grads):
        if forward_ad._current_level >= 0 and any(g is not None and forward_ad.unpack_dual(g).tangent is not None for g in grads):
            TokenFunction.jvp(ctx)
        return guarded(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)
    return run


def same_device(x, *others):
    if not x.is_cuda:
        raise NotImplementedError("rt_pose_amd has no CPU path")
    index = x.get_device()
    for t in others:
        if t is not None and t.get_device() != index:
            raise ValueError("operands on different devices (%s and %s)" % (x.device, t.device))


def like(t):
    """An uninitialised contiguous tensor of t's shape and type."""
    return torch.empty_like(t) if t.is_contiguous() else torch.empty_like(t, memory_format=torch.contiguous_format)


def rows_of(t):
    """[..., n] as [rows, n] with unit stride along the row: a view where there is one, a copy otherwise."""
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    return t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()


def fp8_rows(shape, device, scale_rows=None):
    """An uninitialised 8-bit operand of `shape` (rows of a multiple of 16 bytes in memory) and its scales, one for 128 columns of each row
    (or of `scale_rows` rows)."""
    *lead, n = shape
    wide = -(-n // 16) * 16
    q = torch.empty((*lead, wide), dtype=FP8, device=device)
    scale = torch.empty((*lead, -(-n // 128)) if scale_rows is None else (scale_rows, -(-n // 128)), dtype=torch.float32, device=device)
    return q if wide == n else q[..., :n], scale
