"""The token operators inside a trace: its later calls, of other sizes and layouts, give what the calls by themselves give."""
import pytest
import torch

pytestmark = [pytest.mark.gpu, pytest.mark.filterwarnings("ignore")]


def rnd(*shape, seed, dtype=torch.bfloat16):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


def traced(f, *args):
    with torch.no_grad():
        return torch.jit.trace(f, args, check_trace=False)


def test_cross_attention():
    from rt_pose_amd.attention import cross_attention
    make = lambda b, sq, sk: [rnd(b, n, h, 64, seed=n + h) for n, h in ((sq, 4), (sk, 2), (sk, 2))]
    call = lambda q, k, v, n, m: cross_attention(q, k, v, key_lens=n, key_mask=m)
    lens = torch.tensor([30, 7, 0], device="cuda")
    f = traced(call, *make(2, 3, 20), lens[:2], torch.ones(2, 20, dtype=torch.bool, device="cuda"))
    for b, sq, sk in ((3, 1, 300), (2, 70, 40), (2, 3, 20)):
        q, k, v = make(b, sq, sk)
        m = torch.rand(b, sk, generator=torch.Generator().manual_seed(sk)).cuda() < 0.8
        for t in (q, q.transpose(1, 2).contiguous().transpose(1, 2), torch.cat((q, q), 3)[..., 4:68]):
            assert torch.equal(f(t, k, v, lens[:b], m), call(t, k, v, lens[:b], m))
        leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
        grads = [torch.autograd.grad(g(*leaves, lens[:b], m), leaves, q) for g in (f, call)]
        assert all(torch.equal(a, c) for a, c in zip(*grads))


def test_8_bit_serving():
    from rt_pose_amd.fp8 import matmul_fp8, quantize_fp8
    from rt_pose_amd.rmsnorm import add_rms_norm_fp8
    w, g = rnd(90, 200, seed=1), rnd(200, seed=2, dtype=torch.float32)
    b, sb = quantize_fp8(w, (128, 128))

    def call(x, r):
        q, scale, s = add_rms_norm_fp8(x, r, g)
        return matmul_fp8(q, scale, b, sb), s, *quantize_fp8(x)
    f = traced(call, rnd(3, 200, seed=3), rnd(3, 200, seed=4))
    for rows in (1, 8, 300):
        x, r = rnd(rows, 200, seed=rows), rnd(200, rows, seed=rows + 1).t()
        for u, v in zip(f(x, r), call(x, r)):
            assert torch.equal(u.float(), v.float())


def test_8_bit_operands_that_are_copied():
    from rt_pose_amd.fp8 import _operand, matmul_fp8
    every = torch.arange(256, dtype=torch.uint8, device="cuda").repeat(3, 2).view(torch.float8_e4m3fn)     # every byte, NaN too
    for q in (every[:, 1:300], every[:, ::3], every.t()):
        own, wide = _operand(q, "a")
        assert own.data_ptr() != q.data_ptr() and torch.equal(own[:, :q.shape[1]].contiguous().view(torch.uint8), q.contiguous().view(torch.uint8))
    some = rnd(6, 400, seed=5, dtype=torch.float32).to(torch.float8_e4m3fn)
    scale = lambda n, k: torch.rand(n, -(-k // 128), generator=torch.Generator().manual_seed(k)).cuda()
    f = traced(matmul_fp8, some[:2, :40], scale(2, 40), some[:, :40], scale(6, 40))
    for a, b in ((some[:, 3:333], some[:4, 1:331]), (some[:, ::3][:, :133], some[:, 1::3])):
        args = a, scale(a.shape[0], a.shape[1]), b, scale(b.shape[0], b.shape[1])
        assert torch.equal(f(*args), matmul_fp8(*args))


def test_norms():
    from rt_pose_amd.rmsnorm import add_rms_norm, rms_norm
    w = rnd(200, seed=1).requires_grad_(True)
    f, g = traced(rms_norm, rnd(3, 200, seed=2), w), traced(add_rms_norm, rnd(3, 200, seed=2), rnd(3, 200, seed=3), w)
    for rows in (1, 300):
        x, r = rnd(rows, 200, seed=rows).requires_grad_(True), rnd(200, rows, seed=rows + 1).t().requires_grad_(True)
        for a, b in ((torch.autograd.grad(f(x, w), (x, w), r), torch.autograd.grad(rms_norm(x, w), (x, w), r)),
                     (torch.autograd.grad(g(x, r, w), (x, r, w), (r, x)), torch.autograd.grad(add_rms_norm(x, r, w), (x, r, w), (r, x)))):
            assert all(torch.equal(u, v) for u, v in zip(a, b))
