"""The token operators where offsets pass 32 bits: long caches, many rows.  Every part that stands behind the 2^31st element is compared with the
same rows taken by themselves, or with 64 bits."""
import pytest
import torch

from tests import test_gpu_cross_attention as attn
from tests import test_gpu_matmul_fp8 as mm

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def test_norm_and_quantising():
    from rt_pose_amd.fp8 import quantize_fp8
    from rt_pose_amd.rmsnorm import add_rms_norm, add_rms_norm_fp8
    rows, h = 2 ** 17 + 5, 16384                                          # 2^31 elements and some
    x = torch.empty(rows, h, dtype=BF, device="cuda")
    x.view(torch.int16).random_(0x3C00, 0x4000)                           # bf16 from 2^-7 to 2
    w = torch.rand(h, device="cuda")
    end = x[-6:].clone()

    def same(big, small):
        assert torch.equal(big[-6:].contiguous().view(torch.uint8), small.contiguous().view(torch.uint8))
    for a, b in zip(add_rms_norm_fp8(x, x, w), add_rms_norm_fp8(end, end, w)):
        same(a, b)
    for block in ((1, 128), (128, 128)):
        q, s = quantize_fp8(x[3:] if block[0] == 128 else x, block)       # 2^17 + 2 rows: the last two of them are a block by themselves
        q2, s2 = quantize_fp8(end[-2:] if block[0] == 128 else end, block)
        n = q2.shape[0]
        assert torch.equal(q[-n:].view(torch.uint8), q2.view(torch.uint8)) and torch.equal(s[-s2.shape[0]:], s2)
    q, s = quantize_fp8(x.t())                                            # the last rows are the end of the columns in memory
    q2, s2 = quantize_fp8(x[2 ** 17:].t())
    assert torch.equal(q[:, 2 ** 17:].contiguous().view(torch.uint8), q2.contiguous().view(torch.uint8)) and torch.equal(s[:, -1:], s2)
    del q, s
    x.requires_grad_(True)
    end.requires_grad_(True)
    y, stream = add_rms_norm(x, x.detach(), w)
    y2, stream2 = add_rms_norm(end, end.detach(), w)
    same(y, y2)
    same(stream, stream2)
    (g,) = torch.autograd.grad((y, stream), x, (y.detach(), stream.detach()))
    (g2,) = torch.autograd.grad((y2, stream2), end, (y2.detach(), stream2.detach()))
    same(g, g2)


@pytest.mark.parametrize("m,n,k", [(2 ** 19 + 77, 80, 4096 + 16), (2 ** 20 + 300, 2048 + 8, 48)])
def test_product(m, n, k):
    from rt_pose_amd.fp8 import FP8, matmul_fp8
    b, sb = mm.operand(n, k, True, 1)
    tail, s_tail = mm.operand(400, k, False, 2)
    a = torch.zeros(m, k, dtype=torch.uint8, device="cuda")
    sa = torch.zeros(m, s_tail.shape[1], device="cuda")
    a[-400:].copy_(tail.view(torch.uint8))
    sa[-400:].copy_(s_tail)
    out = matmul_fp8(a.view(FP8), sa, b, sb)
    mm.check(out[-400:], tail, s_tail, b, sb, True)
    assert not bool(out[:m - 400].any())
    turned = matmul_fp8(tail, s_tail, a[-n:].view(FP8), sa[-n:]) if n < 400 else None      # rows with a scale each, from far behind the start
    if turned is not None:
        mm.check(turned, tail, s_tail, a[-n:].view(FP8), sa[-n:], False)


@pytest.mark.parametrize("sq", [1, 40, 150])
def test_long_cache_of_wide_tokens(sq):
    """Tokens 1024 elements apart, of which the operator reads two heads' worth of eight: 2.2 million of them, and a second batch entry behind."""
    from rt_pose_amd.attention import cross_attention
    b, sk, d, step = 2, 2200000, 8, 1024
    big = torch.zeros(b * sk * step, dtype=BF, device="cuda").view(b, sk, 1, step)
    g = torch.Generator(device="cuda").manual_seed(3)
    big[..., :2 * d] = torch.randn(b, sk, 1, 2 * d, device="cuda", generator=g).to(BF)
    k, v = (big[..., i * d:(i + 1) * d].detach().requires_grad_(True) for i in range(2))
    q = torch.randn(b, sq, 1, d, device="cuda", generator=g).to(BF).requires_grad_(True)
    do = torch.randn(b, sq, 1, d, device="cuda", generator=g).to(BF)
    lens = torch.tensor([100, sk])
    o = cross_attention(q, k, v, lens.cuda())
    got = (o, *torch.autograd.grad(o, (q, k, v), do))
    short = torch.cat((k[:1, :100], k[1:, -100:])), torch.cat((v[:1, :100], v[1:, -100:]))
    alone = cross_attention(q[:1], *(t[:1].detach().contiguous() for t in short))
    assert torch.allclose(o[:1].float(), alone.float(), rtol=2 ** -7, atol=2 ** -12)
    Q, K, V, D = (t[1, :, 0].detach().double() for t in (q, k, v, do))
    s = Q @ K.t() * d ** -0.5
    p = torch.softmax(s, 1)
    want = p @ V
    # bounds as in test_gpu_cross_attention, the sums over all keys at n = sk
    u, F = 2.0 ** -8, 2.0 ** -24
    E = 2 * (d + 8) * F * (float((Q.abs() @ K.abs().t()).max()) * d ** -0.5 + 1) + 2.0 ** -20
    assert bool(((o[1, :, 0].double() - want).abs() <= (2 * (E + u) + sk * F) * (p @ V.abs()) + u * want.abs()).all())
    dv = p[:, -100:].t() @ D
    tol = (E + u + sq * F + sk * F) * (p[:, -100:].t() @ D.abs()) + u * dv.abs() + 2.0 ** -126
    assert bool(((got[3][1, -100:, 0].double() - dv).abs() <= tol).all())
    assert not bool(got[3][0, 100:].any()) and not bool(got[2][0, 100:].any()) and bool(got[2][1, -100:].any())


def test_gradients_behind_the_32nd_bit():
    """dk and dv of over 2^31 elements each: a few rows and many; the last keys against the same keys in a cache of their own."""
    from rt_pose_amd.attention import cross_attention
    sk, hkv, d = 2 ** 22 + 200, 8, 64
    g = torch.Generator(device="cuda").manual_seed(4)
    tail = torch.randn(1, 200, hkv, d, device="cuda", generator=g).to(BF)
    k = torch.zeros(1, sk, hkv, d, dtype=BF, device="cuda")
    k[:, -200:] = tail
    mask = torch.zeros(1, sk, dtype=torch.bool, device="cuda")
    mask[:, -200:] = True
    for sq in (2, 70):
        q, do = (torch.randn(1, sq, hkv, d, device="cuda", generator=g).to(BF) for _ in range(2))
        q.requires_grad_(True)
        big, own = k.detach().requires_grad_(True), tail.detach().requires_grad_(True)
        o = cross_attention(q, big, big, None, mask)
        dq, dk = torch.autograd.grad(o, (q, big), do)
        want = attn.reference(q, own, own, attn.seen_of(1, 200, None, None), d ** -0.5, do)
        attn.check((o, dq), want[:2])
        (value, tol), (v2, t2) = want[2], want[3]                          # k and v are one tensor: the gradients add, rounded once more
        total = value + v2
        assert bool(((dk[:, -200:].double() - total).abs() <= tol + t2 + 2.0 ** -8 * (total.abs() + tol + t2)).all())
        assert not bool(dk[:, :-200].any())
        del o, dq, dk, big


@pytest.mark.parametrize("dtype,h", [(torch.float16, 777), (torch.float32, 1031), (BF, 136)])
def test_outputs_larger_than_the_caches_hold(dtype, h):
    from rt_pose_amd.rmsnorm import add_rms_norm, add_rms_norm_fp8, rms_norm
    rows = (2 ** 28 + 2 ** 20) // (h * torch.finfo(dtype).bits // 8)
    x = torch.randn(rows, h, device="cuda", generator=torch.Generator(device="cuda").manual_seed(h)).to(dtype)
    w = torch.rand(h, device="cuda")
    some = torch.cat((x[:33], x[rows // 2:rows // 2 + 40], x[-41:]))
    pick = lambda t: torch.cat((t[:33], t[rows // 2:rows // 2 + 40], t[-41:]))
    for a, b in ((rms_norm(x, w), rms_norm(some, w)), *zip(add_rms_norm(x, x, w), add_rms_norm(some, some, w)),
                 *zip(add_rms_norm_fp8(x, x, w), add_rms_norm_fp8(some, some, w))):
        assert torch.equal(pick(a.view(torch.uint8) if a.dtype.itemsize == 1 else a), b.view(torch.uint8) if b.dtype.itemsize == 1 else b)
