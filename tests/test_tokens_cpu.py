"""Refusals of the token operators' entry points, without a GPU: nothing computes on the CPU, and the C entries check their arguments before
they launch."""
import ctypes as C

import pytest
import torch

from rt_pose_amd import _lib

SHAPE, UNSUPPORTED, ALIGN = -1, -2, -4
P = C.c_void_p


def test_there_is_no_cpu_path():
    from rt_pose_amd.fp8 import matmul_fp8, quantize_fp8
    from rt_pose_amd.rmsnorm import RMSNorm, add_rms_norm, add_rms_norm_fp8, rms_norm
    x, w = torch.zeros(2, 128), torch.ones(128)
    for call in (lambda: rms_norm(x, w), lambda: add_rms_norm(x, x, w), lambda: add_rms_norm_fp8(x, None, w), lambda: RMSNorm(128)(x),
                 lambda: quantize_fp8(x), lambda: matmul_fp8(x.to(torch.float8_e4m3fn), x[:, :1], x.to(torch.float8_e4m3fn), x[:1, :1])):
        with pytest.raises(NotImplementedError):
            call()


def test_norm_entries_check_before_they_launch():
    lib = _lib.load()
    a = P(4096)     # never read: every call below is refused, or has no rows
    assert lib.rtp_rmsnorm_forward(a, 8, None, 0, a, 0, a, None, 0, 8, 0, 1e-6, None) == 0
    assert lib.rtp_rmsnorm_forward(a, 8, None, 0, a, 0, a, None, -1, 8, 0, 1e-6, None) == SHAPE
    assert lib.rtp_rmsnorm_forward(a, 8, None, 0, a, 0, a, None, 1, 0, 0, 1e-6, None) == SHAPE
    assert lib.rtp_rmsnorm_forward(a, 8, None, 0, a, 0, a, None, 1, 16385, 0, 1e-6, None) == UNSUPPORTED
    assert lib.rtp_rmsnorm_forward(a, 8, None, 0, None, 0, a, None, 1, 8, 0, 1e-6, None) == SHAPE
    assert lib.rtp_rmsnorm_forward(a, 8, a, 8, a, 0, a, None, 1, 8, 0, 1e-6, None) == SHAPE        # a residual without a stream to write
    assert lib.rtp_rmsnorm_forward(a, 8, None, 0, a, 1, a, None, 1, 8, 0, 1e-6, None) == UNSUPPORTED
    assert lib.rtp_rmsnorm_forward(a, 8, None, 0, a, 0, a, None, 1, 8, 7, 1e-6, None) == UNSUPPORTED
    assert lib.rtp_rmsnorm_fp8_forward(a, 8, None, 0, a, 0, a, 8, a, None, 1, 8, 0, 1e-6, None) == SHAPE
    assert lib.rtp_rmsnorm_fp8_forward(a, 8, None, 0, a, 0, a, 24, a, None, 1, 8, 0, 1e-6, None) == ALIGN
    assert lib.rtp_rmsnorm_fp8_forward(a, 8, None, 0, a, 0, P(4104), 16, a, None, 1, 8, 0, 1e-6, None) == ALIGN
    assert lib.rtp_rmsnorm_backward(a, 8, a, 0, None, 8, None, 0, a, a, a, 1, 8, 0, 1e-6, None) == SHAPE
    assert lib.rtp_rmsnorm_backward(a, 8, a, 0, a, 8, None, 0, a, a, a, 0, 8, 0, 1e-6, None) == SHAPE
    assert lib.rtp_rmsnorm_backward_slots(0, 8) == 0 and lib.rtp_rmsnorm_backward_slots(1, 8) == 1
    for rows in (1, 17, 20000, 10 ** 6):
        for h in (1, 128, 129, 2048, 2049, 16384):
            assert 1 <= lib.rtp_rmsnorm_backward_slots(rows, h) <= min(rows, 512)


def test_8_bit_entries_check_before_they_launch():
    lib = _lib.load()
    a = P(4096)
    assert lib.rtp_quantize_fp8(a, 8, 0, a, 16, a, 0, 8, 0, 0, None) == 0
    assert lib.rtp_quantize_fp8(a, 8, 0, a, 16, a, 1, 0, 0, 0, None) == SHAPE
    assert lib.rtp_quantize_fp8(a, 8, 0, a, 16, a, 1, 17, 0, 0, None) == SHAPE
    assert lib.rtp_quantize_fp8(a, 8, 0, a, 24, a, 1, 8, 0, 0, None) == ALIGN
    assert lib.rtp_quantize_fp8(a, 8, 0, a, 16, a, 1, 8, 0, 5, None) == UNSUPPORTED
    assert lib.rtp_quantize_fp8(a, 8, 0, a, 16, a, 2 ** 45, 8, 1, 0, None) == SHAPE
    mm = lambda **k: lib.rtp_matmul_fp8(*(dict(dict(a=a, lda=128, sa=a, b=a, ldb=128, sb=a, sq=1, out=a, m=2, n=2, k=128, t=2, s=None), **k).values()))
    assert mm(m=0) == 0 and mm(n=0) == 0
    assert mm(k=0) == SHAPE and mm(m=-1) == SHAPE and mm(a=None) == SHAPE and mm(lda=112) == SHAPE and mm(k=129) == SHAPE
    assert mm(lda=136) == ALIGN and mm(b=P(4097)) == ALIGN and mm(t=3) == UNSUPPORTED
    assert mm(m=2 ** 31 - 1, n=2 ** 31 - 1) == SHAPE
