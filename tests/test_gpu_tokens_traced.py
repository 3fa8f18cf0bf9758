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
