"""Calls of the token operators' C entries that the Python layer does not make."""
import ctypes as C

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("sq", [1, 70])
@pytest.mark.parametrize("lse", [False, True])
def test_cross_attention_without_keys_beside_a_mask(sq, lse):
    """No keys, but a mask's and the keys' buffers: zeros."""
    from rt_pose_amd import _lib, attention
    q, k = (torch.ones(2, n, 4, 32, dtype=torch.bfloat16, device="cuda") for n in (sq, 8))
    mask = torch.ones(2, 8, dtype=torch.bool, device="cuda")
    a = attention._operands(q, k, k, None, mask, 0.5)
    a.sk = 0
    lib = _lib.load()
    n = lib.rtp_xattn_workspace_bytes(C.byref(a), 0)
    assert n == 0
    o, lo = torch.full_like(q, 7.0), torch.full_like(q, 7.0) if lse else None
    stat = torch.zeros(q.shape[:3].numel() + 64, device="cuda") if lse else None
    p = lambda t: None if t is None else t.data_ptr()
    assert lib.rtp_xattn_forward(C.byref(a), p(o), p(lo), p(stat), None, 0, torch.cuda.current_stream().cuda_stream) == 0
    assert float(o.abs().sum()) == 0
    if lse:
        assert float(lo.abs().sum()) == 0 and bool((stat[:q.shape[:3].numel()] == float("inf")).all())
