"""Marshalling shared by the token operators (rmsnorm.py, fp8.py, attention.py)."""
import ctypes as C

import torch

DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}   # RTP_DT_* of include/rtp.h
FP8 = torch.float8_e4m3fn


def p(t):
    return C.c_void_p(t.data_ptr()) if t is not None else None


def stream_of(t):
    return C.c_void_p(torch.cuda.current_stream(t.device).cuda_stream)


def on_device(t):
    """Launches go to the tensor's device, whichever is current."""
    return torch.cuda.device(t.device)


def same_device(x, *others):
    if not x.is_cuda:
        raise NotImplementedError("rt_pose_amd has no CPU path")
    for t in others:
        if t is not None and t.device != x.device:
            raise ValueError("operands on different devices (%s and %s)" % (x.device, t.device))


def rows_of(t):
    """[..., n] as [rows, n] with unit stride along the row: a view where there is one, a copy otherwise."""
    t = t.reshape(-1, t.shape[-1])
    return t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()


def fp8_rows(shape, device, scale_rows=None):
    """An uninitialised 8-bit operand of `shape` (rows of a multiple of 16 bytes in memory) and its scales, one for 128 columns of each row
    (or of `scale_rows` rows)."""
    *lead, n = shape
    q = torch.empty((*lead, -(-n // 16) * 16), dtype=torch.uint8, device=device).view(FP8)[..., :n]
    scale = torch.empty((*lead, -(-n // 128)) if scale_rows is None else (scale_rows, -(-n // 128)), dtype=torch.float32, device=device)
    return q, scale
