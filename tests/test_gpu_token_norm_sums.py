"""The gradients of the norm where many rows are summed: dw and dx against 64 bits with more rows than the kernel has partial rows times row groups, and
partial rows that one pass of the last sum does not cover.

dw, f = 2^-24: a term dy s rho has two roundings and rho's own error: a lane's sum of up to 8 chunks' squares, six steps over the wave, eight waves,
halved by the root, and three roundings more (26 at most).  A group adds its R rows one after the other, the G groups of a workgroup are added,
every 64th of the S partial rows, and six steps of a tree: R + G + S / 64 + 6 roundings of the sum of magnitudes."""
import pytest
import torch

from tests.test_gpu_token_norm import TYPES, U, close, half, rnd

pytestmark = pytest.mark.gpu

ROWS = [(20001, 100), (17000, 8), (16385, 5), (4500, 300), (9001, 777), (5003, 2000), (1301, 2600), (1300, 4100), (700, 12345), (515, 16384),
        (387, 640), (261, 1024), (1030, 64), (130, 5001)]       # the last four: 65 to 130 partial rows


@pytest.mark.parametrize("w32", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,h", ROWS)
def test_gradients_of_many_rows(rows, h, dtype, w32):
    from rt_pose_amd import _lib
    from rt_pose_amd.rmsnorm import add_rms_norm, rms_norm
    slots = _lib.load().rtp_rmsnorm_backward_slots(rows, h)
    assert slots > 64
    eps = 1e-5
    x, r = rnd(rows, h, seed=1, dtype=dtype).requires_grad_(True), rnd(rows, h, seed=2, dtype=dtype, scale=3.0).requires_grad_(True)
    w = (1 + rnd(h, seed=3, dtype=torch.float32, scale=0.3)).to(torch.float32 if w32 else dtype).requires_grad_(True)
    dy, ds = rnd(rows, h, seed=4, dtype=dtype), rnd(rows, h, seed=5, dtype=dtype)
    y, s = add_rms_norm(x, r, w, eps)
    dx, dr, dw = torch.autograd.grad((y, s), (x, r, w), (dy, ds))
    assert torch.equal(dx, dr)
    s64, w64 = s.detach().double(), w.detach().double()
    root = torch.sqrt((s64 * s64).mean(-1, keepdim=True) + eps)
    g, xh = dy.double() * w64, s64 / root
    own = (g - xh * (g * xh).mean(-1, keepdim=True)) / root
    mag = (g.abs() + xh.abs() * (g * xh).abs().mean(-1, keepdim=True)) / root
    close(dx, own + ds.double(), (own + ds.double()).abs() * half(dtype) + U * (mag + ds.double().abs()), "dx")
    groups = 16 if h <= 128 else 4 if h <= 2048 else 1
    adds = -(-rows // (slots * groups)) + groups + -(-slots // 64) + 6
    term = dy.double() * xh
    bound = lambda dw64: dw64.abs() * half(w.dtype) + (adds + 2 + 26) * 2.0 ** -24 * term.abs().sum(0)
    close(dw, term.sum(0), bound(term.sum(0)), "dw")
    z = s.detach().requires_grad_(True)                       # the same rows without a residual
    gz, gw = torch.autograd.grad(rms_norm(z, w, eps), (z, w), dy)
    close(gz, own, own.abs() * half(dtype) + U * mag, "dx alone")
    assert torch.equal(gw, dw)


def test_every_row_counts_once():
    """A gradient in one row alone gives that row's share of dw, wherever the row stands: whole numbers, exact in any order."""
    from rt_pose_amd.rmsnorm import rms_norm
    for rows, h in ((20001, 100), (9001, 777), (1301, 2600), (700, 12345)):
        x = torch.ones(rows, h, device="cuda")
        w = torch.ones(h, device="cuda", requires_grad=True)
        share = torch.randint(-8, 9, (rows, 1), generator=torch.Generator().manual_seed(h)).float().cuda()
        (dw,) = torch.autograd.grad(rms_norm(x, w, 0.0), w, share.expand(rows, h).contiguous())
        assert torch.equal(dw, share.sum().expand(h))
