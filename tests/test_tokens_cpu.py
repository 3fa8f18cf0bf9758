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
            assert 1 <= lib.rtp_rmsnorm_backward_slots(rows, h) <= min(rows, 1024)


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


def test_cross_attention_has_no_cpu_path():
    from rt_pose_amd.attention import cross_attention
    q = torch.zeros(1, 2, 4, 32, dtype=torch.bfloat16)
    with pytest.raises(NotImplementedError):
        cross_attention(q, q, q)


def attn(**k):
    a = _lib.RtpXattn()
    for n in ("q", "k", "v"):
        setattr(a, n, 4096)
    for n, v in dict(dict(b=2, sq=3, sk=5, hq=4, hkv=2, d=64, dtype=2, scale=0.125, q_bs=768, q_ss=256, q_hs=64, k_bs=640, k_ss=128, k_hs=64,
                          v_bs=640, v_ss=128, v_hs=64), **k).items():
        setattr(a, n, v)
    return a


def test_cross_attention_entries_check_before_they_launch():
    lib = _lib.load()
    o = P(4096)
    size = lambda back=0, **k: lib.rtp_xattn_workspace_bytes(C.byref(attn(**k)), back)
    fwd = lambda o_lo=None, lse=None, ws=None, n=0, **k: lib.rtp_xattn_forward(C.byref(attn(**k)), o, o_lo, lse, ws, n, None)
    bwd = lambda dq=o, dk=o, dv=o, ws=o, n=1 << 40, os=64, **k: lib.rtp_xattn_backward(C.byref(attn(**k)), o, o, o, o, 768, 256, os, dq, dk, dv, ws, n, None)
    assert size() == 0 and size(1) > 0
    assert fwd(b=0) == 0 and fwd(sq=0) == 0
    for bad in (dict(b=-1), dict(sq=-1), dict(sk=-1), dict(hq=3), dict(hkv=0), dict(d=0), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")),
                dict(scale=float("inf")), dict(sk=2 ** 30 + 1), dict(sq=2 ** 30, hq=64)):
        assert fwd(**bad) == SHAPE and size(**bad) == -1 and bwd(**bad) == SHAPE
    for bad in (dict(d=12), dict(d=136), dict(dtype=0), dict(dtype=3)):
        assert fwd(**bad) == UNSUPPORTED and bwd(**bad) == UNSUPPORTED
    for bad in (dict(q=4100), dict(q_hs=4), dict(k_ss=130), dict(v_bs=641)):
        assert fwd(**bad) == ALIGN and bwd(**bad) == ALIGN
    assert fwd(q=None) == SHAPE and fwd(k=None) == SHAPE and fwd(o_lo=o) == SHAPE and fwd(lse=o) == SHAPE
    assert fwd(key_mask=4096, ws=None, n=0) == SHAPE                      # a mask needs a workspace
    assert bwd(os=60) == ALIGN and bwd(ws=P(4112)) == ALIGN and bwd(n=8) == SHAPE and bwd(dk=None) == SHAPE and bwd(ws=None) == SHAPE
    assert bwd(b=0) == SHAPE and bwd(sk=0) == SHAPE


def test_workspace_is_sized_for_every_cut():
    """The cut of the work depends on sizes alone; its partial results stay a fraction of what the pass reads and writes anyway or small."""
    lib = _lib.load()
    for b in (1, 3, 16):
        for sq in (1, 15, 40, 700, 5000):
            for sk in (0, 1, 64, 5000, 10 ** 6):
                for hq, hkv in ((1, 1), (8, 2), (12, 12)):
                    for back in (0, 1):
                        n = lib.rtp_xattn_workspace_bytes(C.byref(attn(b=b, sq=sq, sk=sk, hq=hq, hkv=hkv)), back)
                        assert 0 <= n < 2 ** 33


def test_sizes_that_no_launch_can_count_are_refused():
    """A launch counts its threads in 32 bits; what would pass that is refused before anything is read."""
    lib = _lib.load()
    a = P(4096)
    for rows, h in ((2 ** 28, 8), (2 ** 26, 200), (2 ** 24, 4096), (2 ** 31, 8)):
        assert lib.rtp_rmsnorm_forward(a, h, None, 0, a, 0, a, None, rows, h, 0, 1e-6, None) == SHAPE
        assert lib.rtp_rmsnorm_fp8_forward(a, h, None, 0, a, 0, a, 4096, a, None, rows, h, 0, 1e-6, None) == SHAPE
    for rows, cols, square, turned in ((2 ** 30, 8, 0, 0), (2 ** 31, 8, 1, 0), (2 ** 28, 8, 0, 1), (2 ** 28, 8, 1, 1), (1, 2 ** 30 + 1, 0, 0)):
        assert lib.rtp_quantize_fp8(a, cols, turned, a, 2 ** 31, a, rows, cols, square, 0, None) == SHAPE
    for m, n in ((2 ** 30 + 1, 1), (1, 2 ** 30 + 1), (1, 2 ** 29), (2 ** 20, 2 ** 20)):
        assert lib.rtp_matmul_fp8(a, 16, a, a, 16, a, 1, a, m, n, 16, 2, None) == SHAPE
    assert lib.rtp_matmul_fp8(a, 2 ** 22 + 16, a, a, 16, a, 1, a, 2, 2, 16, 2, None) == SHAPE
    size = lambda back=0, **k: lib.rtp_xattn_workspace_bytes(C.byref(attn(**k)), back)
    for bad in (dict(b=2 ** 24, hkv=1, hq=1), dict(b=2 ** 20, sk=2 ** 16), dict(b=2 ** 10, sq=2 ** 18, hq=2, hkv=2), dict(scale=2.5e38), dict(b=2 ** 30, hkv=64, hq=64)):
        assert size(**bad) == -1 and size(1, **bad) == -1
