"""cross_attention with many rows, where no waves share them (four groups of 32 rows a workgroup, two sub-tiles of keys a wave): against 64 bits, with
the bounds of test_gpu_cross_attention."""
import ctypes as C

import pytest
import torch

from tests.test_gpu_cross_attention import case, check, reference, rnd, seen_of

pytestmark = pytest.mark.gpu


def row_waves(q, k):
    """how many waves of a workgroup share rows in a call of these sizes"""
    from rt_pose_amd import _lib, attention
    return _lib.load().rtp_xattn_row_waves(C.byref(attention._operands(q, k, k, None, None, 1.0)))


def steps(n, sk):
    """lengths of n batch entries: one without keys, one with all, the others between"""
    return [0, sk, *((7 * i * i + 3 * i + 1) % (sk + 1) for i in range(n - 2))]


SHAPES = [  # b, sq, sk, hq, hkv, d, lengths, share of keys that count
    (64, 70, 200, 16, 16, 32, True, 0.8),
    (16, 1030, 130, 8, 8, 64, True, None),
    (16, 515, 70, 16, 8, 128, False, 0.7),
    (33, 1000, 90, 4, 4, 96, False, None),
    (128, 40, 65, 24, 8, 72, True, 0.9),            # groups of three heads: no step of a staged tile is a whole number of tokens
    (2, 8200, 40, 8, 8, 64, True, None),
    (64, 65, 1, 16, 16, 8, False, None),
    (128, 33, 321, 16, 8, 40, True, None),
    (171, 128, 64, 6, 6, 128, False, None),
    (37, 500, 129, 7, 7, 16, True, 0.5),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s[:6])))
def test_forward_and_gradients(shape, dtype):
    from rt_pose_amd.attention import cross_attention
    b, sq, sk, hq, hkv, d, lens, share = shape
    q, k, v, do, lens, mask = case(b, sq, sk, hq, hkv, d, dtype, steps(b, sk) if lens else None, share, seed=b)
    assert row_waves(q, k) == 1
    L = None if lens is None else lens.cuda()
    want = reference(q, k, v, seen_of(b, sk, lens, mask), d ** -0.5, do)
    with torch.no_grad():
        check([cross_attention(q, k, v, L, mask)], want[:1])
    o = cross_attention(q, k, v, key_lens=L, key_mask=mask)
    grads = torch.autograd.grad(o, (q, k, v), do)
    check([o, *grads], want)
    o2 = cross_attention(q, k, v, key_lens=L, key_mask=mask)
    assert all(torch.equal(a, c) for a, c in zip((o, *grads), (o2, *torch.autograd.grad(o2, (q, k, v), do))))
    (gv,) = torch.autograd.grad(cross_attention(q.detach(), k.detach(), v, L, mask), v, do)      # no gradient of q: delta by itself
    (gk,) = torch.autograd.grad(cross_attention(q.detach(), k, v.detach(), L, mask), k, do)
    check([o, grads[0], gk, gv], want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_what_masked_keys_hold_does_not_matter(dtype):
    from rt_pose_amd.attention import cross_attention
    b, sk = 64, 150
    q, k, v, do, lens, mask = case(b, 66, sk, 16, 16, 64, dtype, steps(b, sk), 0.6, seed=11)
    assert row_waves(q, k) == 1
    L, seen = lens.cuda(), seen_of(b, sk, lens, mask)
    outs = []
    for fill in (0.0, float("nan"), float("inf"), torch.finfo(dtype).min):
        kk, vv = (torch.where(seen[:, :, None, None], x.detach(), fill).requires_grad_(True) for x in (k, v))
        o = cross_attention(q, kk, vv, L, mask)
        outs.append((o, *torch.autograd.grad(o, (q, kk, vv), do)))
    for other in outs[1:]:
        assert all(torch.equal(a, c) for a, c in zip(outs[0], other))
    o, dq, dk, dv = outs[1]
    assert float(o[0].abs().sum()) == 0 and float(dq[0].abs().sum()) == 0
    assert float(dk[~seen].abs().sum()) == 0 and float(dv[~seen].abs().sum()) == 0


@pytest.mark.parametrize("sk,qk,vs,dos", [(3000, 1.0, 1.0, 0.02), (4, 0.01, 3.0, 2e4), (300, 0.01, 3.0, 2e4)])
def test_gradients_at_both_ends_of_fp16(sk, qk, vs, dos):
    """p and ds far below fp16's normal range, and ds beyond its largest value: the factor of a row falls while both sub-tiles of keys are under way."""
    from rt_pose_amd.attention import cross_attention
    b, sq, h, d = 64, 66, 16, 64
    q, do = rnd(b, sq, h, d, seed=1, dtype=torch.float16, scale=qk).requires_grad_(True), rnd(b, sq, h, d, seed=2, dtype=torch.float16, scale=dos)
    k, v = (rnd(b, sk, h, d, seed=3 + i, dtype=torch.float16, scale=z).requires_grad_(True) for i, z in enumerate((qk, vs)))
    do = do.clamp(-6e4, 6e4)
    assert row_waves(q, k) == 1
    o = cross_attention(q, k, v)
    got = (o, *torch.autograd.grad(o, (q, k, v), do))
    assert all(bool(torch.isfinite(x).all()) for x in got[1:3])
    for x, (y, tol) in zip(got, reference(q, k, v, torch.ones(b, sk, dtype=torch.bool, device="cuda"), d ** -0.5, do)):
        x, fits, over = x.detach().double(), y.abs() + tol < 65504, y.abs() - tol >= 65520          # from 65520 on the nearest value is infinity
        assert float(((x - y).abs() - tol)[fits].max()) <= 0
        assert torch.equal(x[over], torch.copysign(torch.full_like(y, float("inf")), y)[over])


def test_large_scores_and_uneven_ones():
    """One key takes all; a running maximum that climbs through all tiles."""
    from rt_pose_amd.attention import cross_attention
    b, sq, sk, h, d = 64, 80, 700, 16, 64
    q = rnd(b, sq, h, d, seed=1, dtype=torch.bfloat16, scale=8.0).requires_grad_(True)
    k = (rnd(b, sk, h, d, seed=2, dtype=torch.float32, scale=4.0) * torch.linspace(0.1, 2.0, sk, device="cuda")[None, :, None, None]).to(torch.bfloat16)
    k.requires_grad_(True)
    v, do = rnd(b, sk, h, d, seed=3, dtype=torch.bfloat16).requires_grad_(True), rnd(b, sq, h, d, seed=4, dtype=torch.bfloat16)
    assert row_waves(q, k) == 1
    o = cross_attention(q, k, v)
    want = reference(q, k, v, torch.ones(b, sk, dtype=torch.bool, device="cuda"), d ** -0.5, do)
    for x, (y, tol) in zip((o, *torch.autograd.grad(o, (q, k, v), do)), want):
        assert float(((x.detach().double() - y).abs() - tol).max()) <= 0


def test_strides_and_a_capture():
    from rt_pose_amd.attention import cross_attention
    b, sk = 64, 100
    q, k, v, do, lens, mask = case(b, 66, sk, 32, 16, 32, torch.bfloat16, steps(b, sk), 0.8, seed=7)
    assert row_waves(q, k) == 1
    L = lens.cuda()

    def step(q, k, v, do):
        o = cross_attention(q, k, v, L, mask)
        return [t.detach() for t in (o, *torch.autograd.grad(o, (q, k, v), do))]
    want = step(q, k, v, do)
    heads_first = lambda t: t.detach().transpose(1, 2).contiguous().transpose(1, 2)
    both = torch.stack((k.detach(), v.detach()), 2)
    for qq, kk, vv, dd in ((heads_first(q), heads_first(k), heads_first(v), heads_first(do)), (q.detach(), both[:, :, 0], both[:, :, 1], do)):
        got = step(qq.requires_grad_(True), kk.detach().requires_grad_(True), vv.detach().requires_grad_(True), dd)
        assert all(torch.equal(a, c) for a, c in zip(got, want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(q, k, v, do)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(q, k, v, do)
    for seed in range(3):
        with torch.no_grad():
            q.copy_(rnd(b, 66, 32, 32, seed=seed, dtype=torch.bfloat16))
            L.copy_(torch.tensor(steps(b, sk)).roll(seed))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(out, step(q, k, v, do)))
