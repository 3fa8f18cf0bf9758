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


@pytest.mark.parametrize("rows,h", [(3, 7), (5000, 100), (4200, 777), (600, 4100), (300, 12345)])
def test_norm_gradients_with_a_weight_that_is_not_trained(rows, h):
    """dx alone, by Python and by the C entry without dw and its scratch: the same dx; a dw without its scratch is refused."""
    from rt_pose_amd import _lib
    from rt_pose_amd.rmsnorm import add_rms_norm, rms_norm
    g = torch.Generator().manual_seed(rows)
    x, r, dy, ds = (torch.randn(rows, h, generator=g).to(torch.bfloat16).cuda() for _ in range(4))
    w = torch.rand(h, generator=g).cuda()
    x.requires_grad_(True)
    both = torch.autograd.grad(add_rms_norm(x, r, w.clone().requires_grad_(True)), x, (dy, ds))[0]
    assert torch.equal(torch.autograd.grad(add_rms_norm(x, r, w), x, (dy, ds))[0], both)
    want = torch.autograd.grad(rms_norm(x, w.clone().requires_grad_(True)), x, dy)[0]
    assert torch.equal(torch.autograd.grad(rms_norm(x, w), x, dy)[0], want)
    dx, p, s = torch.empty_like(dy), x.data_ptr, torch.cuda.current_stream().cuda_stream
    entry = lambda dw, part: _lib.load().rtp_rmsnorm_backward(p(), h, w.data_ptr(), 0, dy.data_ptr(), h, None, 0, dx.data_ptr(), dw, part, rows, h, 2, 1e-6, s)
    assert entry(w.data_ptr(), None) == -1
    assert entry(None, None) == 0 and torch.equal(dx, want)


@pytest.mark.parametrize("m,n,k", [(4, 40, 264), (300, 200, 520), (1400, 1300, 384)])
def test_products_that_cancel(m, n, k):
    """Large products of opposite sign beside a small one in each group of eight: an fp32 output is exact, the others within what the instruction
    leaves out."""
    from rt_pose_amd.fp8 import matmul_fp8
    from tests.test_gpu_matmul_fp8 import check
    g = torch.Generator().manual_seed(m)
    a = torch.zeros(m, k)
    a[:, 0::8], a[:, 3::8], a[:, 5::8] = 448.0, -448.0, torch.randint(1, 8, (m, len(range(5, k, 8))), generator=g).float()
    b = torch.ones(n, k)
    b[:, 0::8] = b[:, 3::8] = 448.0
    a, b = (t.to(torch.float8_e4m3fn).cuda() for t in (a, b))
    kb = -(-k // 128)
    for square in (True, False):
        sa, sb = torch.ones(m, kb, device="cuda"), torch.ones(-(-n // 128) if square else n, kb, device="cuda")
        exact = a.double()[:, 5::8].sum(1, keepdim=True).expand(m, n)
        assert torch.equal(matmul_fp8(a, sa, b, sb, torch.float32).double(), exact)
        for t in (torch.bfloat16, torch.float16):
            check(matmul_fp8(a, sa, b, sb, t), a, sa, b, sb, square)
