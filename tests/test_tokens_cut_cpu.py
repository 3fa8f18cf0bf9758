"""How cross attention is cut by sizes: the tests of the kernels reach every cut that real sizes do."""
import ctypes as C

from tests.test_tokens_cpu import attn


def waves(**k):
    from rt_pose_amd import _lib
    return _lib.load().rtp_xattn_row_waves(C.byref(attn(**k)))


def test_the_waves_that_share_rows():
    assert waves(b=2, sq=15, hq=8, hkv=8) == 4 and waves(b=8, sq=1, hq=32, hkv=8) == 4      # up to 32 rows of a key head
    assert waves(b=2, sq=16, hq=8, hkv=4) == 4 and waves(b=2, sq=33, hq=8, hkv=8) == 2
    assert waves(b=1, sq=64, hq=8, hkv=8) == 2 and waves(b=4, sq=2560, hq=8, hkv=8) == 2    # fewer than four workgroups to a CU
    assert waves(b=8, sq=2048, hq=8, hkv=8) == 1 and waves(b=64, sq=70, hq=16, hkv=16) == 1
    assert waves(d=12) == -1 and waves(sk=-1) == -1 and waves(hq=3) == -1


def test_the_shapes_of_the_many_row_tests_are_of_that_cut():
    from tests.test_gpu_cross_attention import SHAPES as shared
    from tests.test_gpu_cross_attention_rows import SHAPES as alone
    sizes = lambda s: dict(zip(("b", "sq", "sk", "hq", "hkv", "d"), s))
    assert all(waves(**sizes(s)) == 1 for s in alone)
    assert {waves(**sizes(s)) for s in shared} == {2, 4}
    assert {(s[5] + 31) // 32 for s in alone} == {1, 2, 3, 4}
