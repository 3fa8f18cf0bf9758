"""cross_attention against a plain implementation in 64 bits, elementwise.

Bounds, u = finfo(type).eps / 2 (half a step), f = 2^-24.  A score is a sum of d fp32 products, scaled and put into an exponential: its error moves
p by at most E = 2 (d + 8) f (max sum_d |q k| scale + 1) + 2^-20 (the hardware's exp2), relative; p is rounded to 16 bits (u) for its product.
  o      (2 (E + u) sum p |v|) + u |o|                          numerator and denominator
  dv     ((E + u) sum p |do|) + u |dv|
  ds     p ((E + u) |dp - delta| + (d + 8) f sum |do v| + sum_d |do| eo + 2 d f sum_d |do| sum p |v|) =: es       eo: o's bound without its rounding,
         2^-16 |o| in its place (what is left of o after its own and its remainder's rounding)
  dq     scale sum es |k| + u |dq|,   dk     scale sum es |q| + u |dk|        sums over n terms in fp32: n f of the sum of magnitudes besides
fp16 besides: 2^-25, half of its smallest step, for the output and, times what it is multiplied by, for p and ds.  bf16 in its place: 2^-126,
below which the hardware's exponential gives zero (p and its products vanish there; a formula in 64 bits goes on to 2^-1022)."""
import pytest
import torch

pytestmark = pytest.mark.gpu
F = 2.0 ** -24


def rnd(*shape, seed, dtype, scale=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype).cuda()


def seen_of(b, sk, lens, mask):
    seen = torch.ones(b, sk, dtype=torch.bool, device="cuda")
    if lens is not None:
        seen &= torch.arange(sk, device="cuda") < lens.cuda()[:, None]
    return seen & mask if mask is not None else seen


def reference(q, k, v, seen, scale, do=None):
    """(value, bound) of o and, with do, of dq, dk, dv"""
    t = q.dtype
    b, sq, hq, d = q.shape
    sk, hkv = k.shape[1:3]
    g = hq // hkv
    u, tiny = torch.finfo(t).eps / 2, (2.0 ** -25 if t == torch.float16 else 2.0 ** -126)
    per_head = lambda x: x.double().transpose(1, 2)
    clear = lambda x: torch.where(seen[:, :, None, None], x.detach().double(), 0.0)
    Q = per_head(q.detach())
    K, V = (per_head(clear(x)).repeat_interleave(g, 1) for x in (k, v))
    s = (Q @ K.transpose(2, 3)) * scale
    s = s.masked_fill(~seen[:, None, None, :], float("-inf"))
    p = torch.exp(s - s.amax(3, keepdim=True).clamp_min(-1e300))
    p = p / p.sum(3, keepdim=True).clamp_min(1e-300)
    E = 2 * (d + 8) * F * (float((Q.abs() @ K.abs().transpose(2, 3)).max()) * scale + 1) + 2.0 ** -20 if sk and sq else 0.0
    n = sk * F
    o, pv = p @ V, p @ V.abs()
    eo = (2 * (E + u) + n) * pv + tiny * V.abs().sum(2, keepdim=True)
    heads = lambda x: x.transpose(1, 2)
    out = [(heads(o), heads(eo + u * o.abs()) + tiny)]
    if do is None:
        return out
    D = per_head(do)
    dp, dpm = D @ V.transpose(2, 3), D.abs() @ V.abs().transpose(2, 3)
    delta = (p * dp).sum(3, keepdim=True)
    ds = p * (dp - delta)
    base = (E + u) * (dp - delta).abs() + (d + 8) * F * dpm + (D.abs() * (eo + 2.0 ** -16 * o.abs() + 2 * d * F * pv)).sum(3, keepdim=True)
    es = p * base + tiny * (dp - delta).abs() + tiny
    fold = lambda x: x.reshape(b, hkv, g, sk, d).sum(2).transpose(1, 2)
    m = sq * g * F
    dq, eq = ds @ K * scale, (es @ K.abs() + n * (ds.abs() @ K.abs())) * scale
    dk, ek = ds.transpose(2, 3) @ Q * scale, (es.transpose(2, 3) @ Q.abs() + m * (ds.abs().transpose(2, 3) @ Q.abs())) * scale
    dv, ev = p.transpose(2, 3) @ D, (E + u + m) * (p.transpose(2, 3) @ D.abs()) + tiny * D.abs().sum(2, keepdim=True)
    out.append((heads(dq), heads(eq) + u * heads(dq).abs() + tiny))
    for x, e in ((dk, ek), (dv, ev)):
        out.append((fold(x), fold(e) + u * fold(x).abs() + tiny))
    return out


def check(got, want):
    for name, x, (y, tol) in zip(("o", "dq", "dk", "dv"), got, want):
        assert x.shape == y.shape, name
        bad = (x.detach().double() - y).abs() - tol
        assert not x.numel() or float(bad.max()) <= 0, "%s: over its bound by %g" % (name, float(bad.max()))
        # the bounds add every error up; the errors themselves scatter: four roundings' worth of the result as a whole
        if float(y.norm()) > 0 and y.numel() > 2000:
            rel = float((x.detach().double() - y).norm() / y.norm())
            assert rel < 4 * torch.finfo(x.dtype).eps / 2, "%s: %g off as a whole" % (name, rel)


def case(b, sq, sk, hq, hkv, d, dtype, lens=None, mask=None, seed=0, scale=None):
    q = rnd(b, sq, hq, d, seed=seed, dtype=dtype, scale=1.5).requires_grad_(True)
    k, v = (rnd(b, sk, hkv, d, seed=seed + i, dtype=dtype).requires_grad_(True) for i in (1, 2))
    do = rnd(b, sq, hq, d, seed=seed + 3, dtype=dtype, scale=0.5)
    lens = None if lens is None else torch.tensor(lens, dtype=torch.int32)
    if mask is not None:
        mask = torch.rand(b, sk, generator=torch.Generator().manual_seed(seed + 4)).cuda() < mask
    return q, k, v, do, lens, mask


SHAPES = [  # b, sq, sk, hq, hkv, d, lens, share of keys that count
    (1, 1, 1, 1, 1, 8, None, None),
    (2, 1, 33, 2, 1, 32, None, None),
    (3, 1, 700, 8, 2, 128, [700, 0, 33], None),
    (2, 15, 1000, 4, 4, 32, [1000, 517], 0.7),
    (2, 15, 100, 6, 2, 40, None, 0.5),
    (1, 33, 64, 1, 1, 64, None, None),
    (2, 50, 257, 3, 3, 96, [256, 257], None),
    (1, 64, 128, 5, 1, 16, None, 0.9),
    (2, 100, 5, 2, 2, 64, [1, 5], None),
    (2, 129, 300, 4, 2, 128, [300, 129], 0.8),
    (1, 700, 65, 2, 1, 72, None, None),
    (1, 1000, 1, 2, 2, 32, None, None),
    (1, 31, 6000, 2, 1, 24, None, 0.95),
    (3, 257, 513, 6, 2, 64, [0, 512, 300], None),
    (1, 2000, 40, 7, 1, 120, [37], None),
    (1, 1, 20000, 1, 1, 64, None, None),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s[:6])))
def test_forward_and_gradients(shape, dtype):
    from rt_pose_amd.attention import cross_attention
    q, k, v, do, lens, mask = case(*shape[:6], dtype, *shape[6:])
    L = None if lens is None else lens.cuda()
    want = reference(q, k, v, seen_of(shape[0], shape[2], lens, mask), shape[5] ** -0.5, do)
    with torch.no_grad():
        check([cross_attention(q, k, v, L, mask)], want[:1])
    o = cross_attention(q, k, v, key_lens=L, key_mask=mask)
    grads = torch.autograd.grad(o, (q, k, v), do)
    check([o, *grads], want)
    o2 = cross_attention(q, k, v, key_lens=L, key_mask=mask)
    for a, c in zip((o, *grads), (o2, *torch.autograd.grad(o2, (q, k, v), do))):
        assert torch.equal(a, c)                          # nothing depends on scheduling


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("sq,sk", [(1, 300), (40, 129), (200, 260)])
def test_what_masked_keys_hold_does_not_matter(sq, sk, dtype):
    from rt_pose_amd.attention import cross_attention
    q, k, v, do, lens, mask = case(3, sq, sk, 4, 2, 64, dtype, [sk, sk // 2, 0], 0.6, seed=11)
    L, seen = lens.cuda(), seen_of(3, sk, lens, mask)
    outs = []
    for fill in (0.0, float("nan"), float("inf"), torch.finfo(dtype).min):
        kk, vv = (torch.where(seen[:, :, None, None], x.detach(), fill).requires_grad_(True) for x in (k, v))
        o = cross_attention(q, kk, vv, L, mask)
        outs.append((o, *torch.autograd.grad(o, (q, kk, vv), do)))
    for other in outs[1:]:
        assert all(torch.equal(a, c) for a, c in zip(outs[0], other))
    o, dq, dk, dv = outs[1]
    assert float(o[2].abs().sum()) == 0 and float(dq[2].abs().sum()) == 0
    assert float(dk[~seen].abs().sum()) == 0 and float(dv[~seen].abs().sum()) == 0
    nobody = torch.zeros(3, sk, dtype=torch.bool, device="cuda")
    o = cross_attention(q, k, v, None, nobody)
    assert float(o.abs().sum()) == 0 and all(float(g.abs().sum()) == 0 for g in torch.autograd.grad(o, (q, k, v), do))


def test_one_key_has_no_gradient_for_the_scores():
    from rt_pose_amd.attention import cross_attention
    q, k, v, do, _, _ = case(2, 70, 1, 2, 1, 64, torch.bfloat16, seed=3)
    o = cross_attention(q, k, v)
    dq, dk, _ = torch.autograd.grad(o, (q, k, v), do)
    assert torch.equal(o, v.expand(2, 70, 2, 64))
    # p = 1 and dp = delta up to fp32 summation in two orders, o's remainder included: (2 d + 8) 2^-24 of the magnitudes, and 2^-16 of o
    bound = (do.double().abs() * v.double().abs()).sum(3, keepdim=True) * (2 * 64 * F + 2.0 ** -16) / 8
    assert bool((dq.double().abs() <= bound * k.double().abs() * 1.01).all())


def test_large_scores_and_uneven_ones():
    """Scores in the hundreds: one key takes all, the others vanish; a running maximum that climbs through all tiles; equal scores."""
    from rt_pose_amd.attention import cross_attention
    b, sq, sk, d = 1, 40, 900, 64
    q = rnd(b, sq, 2, d, seed=1, dtype=torch.bfloat16, scale=8.0).requires_grad_(True)
    k = (rnd(b, sk, 2, d, seed=2, dtype=torch.float32, scale=4.0) * torch.linspace(0.1, 2.0, sk, device="cuda")[None, :, None, None]).to(torch.bfloat16)
    k.requires_grad_(True)
    v, do = rnd(b, sk, 2, d, seed=3, dtype=torch.bfloat16).requires_grad_(True), rnd(b, sq, 2, d, seed=4, dtype=torch.bfloat16)
    seen = torch.ones(b, sk, dtype=torch.bool, device="cuda")
    o = cross_attention(q, k, v)
    for x, (y, tol) in zip((o, *torch.autograd.grad(o, (q, k, v), do)), reference(q, k, v, seen, d ** -0.5, do)):
        assert float(((x.detach().double() - y).abs() - tol).max()) <= 0
    same = torch.zeros(b, sk, 2, d, dtype=torch.bfloat16, device="cuda")
    o = cross_attention(q, same, v.detach())
    check([o], reference(q, same, v, seen, d ** -0.5)[:1])


@pytest.mark.parametrize("sq", [10, 50, 150])
def test_gradients_at_both_ends_of_fp16(sq):
    """p and ds far below fp16's normal range (many keys, small gradients), and ds beyond its largest value (few keys, large ones)."""
    from rt_pose_amd.attention import cross_attention
    for sk, qk, vs, dos in ((20000, 1.0, 1.0, 0.02), (4, 0.01, 3.0, 2e4), (300, 0.01, 3.0, 2e4)):
        n = sq if sk == 20000 else sq // 8
        q, do = rnd(1, n, 2, 64, seed=1, dtype=torch.float16, scale=qk).requires_grad_(True), rnd(1, n, 2, 64, seed=2, dtype=torch.float16, scale=dos)
        k, v = (rnd(1, sk, 2, 64, seed=3 + i, dtype=torch.float16, scale=z).requires_grad_(True) for i, z in enumerate((qk, vs)))
        do = do.clamp(-6e4, 6e4)
        o = cross_attention(q, k, v)
        got = (o, *torch.autograd.grad(o, (q, k, v), do))
        assert all(bool(torch.isfinite(x).all()) for x in got[1:3])
        for x, (y, tol) in zip(got, reference(q, k, v, torch.ones(1, sk, dtype=torch.bool, device="cuda"), 64 ** -0.5, do)):
            fits = y.abs() + tol < 65504
            assert float((((x.detach().double() - y).abs() - tol) * fits).max()) <= 0


@pytest.mark.parametrize("scale", [1e-6, 0.25, 2.0])
def test_scale(scale):
    from rt_pose_amd.attention import cross_attention
    q, k, v, do, _, _ = case(1, 40, 200, 2, 2, 32, torch.float16, seed=5)
    o = cross_attention(q, k, v, scale=scale)
    for x, (y, tol) in zip((o, *torch.autograd.grad(o, (q, k, v), do)),
                           reference(q, k, v, torch.ones(1, 200, dtype=torch.bool, device="cuda"), scale, do)):
        assert float(((x.detach().double() - y).abs() - tol).max()) <= 0


@pytest.mark.parametrize("sq", [1, 90])
def test_strides_types_of_lengths_and_streams(sq):
    from rt_pose_amd.attention import cross_attention
    b, sk, hq, hkv, d = 2, 150, 4, 2, 64
    q, k, v, do, lens, mask = case(b, sq, sk, hq, hkv, d, torch.bfloat16, [150, 60], 0.8, seed=7)
    L = lens.cuda()
    o = cross_attention(q, k, v, L, mask)
    want = (o, *torch.autograd.grad(o, (q, k, v), do))

    def same(q2, k2, v2, do2, L2=L, m2=mask):
        o2 = cross_attention(q2, k2, v2, L2, m2)
        got = (o2, *torch.autograd.grad(o2, (q2, k2, v2), do2))
        assert all(torch.equal(a, c) for a, c in zip(got, want))
    leaf = lambda t: t.detach().requires_grad_(True)
    heads_first = lambda t: leaf(t.detach().transpose(1, 2).contiguous().transpose(1, 2))
    same(heads_first(q), heads_first(k), heads_first(v), heads_first(do).detach())
    both = torch.stack((k.detach(), v.detach()), 2)                       # one tensor of keys and values, as one projection leaves them
    same(q, leaf(both[:, :, 0]), leaf(both[:, :, 1]), do)

    def odd(t):                                                           # rows that start at any multiple of two bytes
        wide = torch.zeros(*t.shape[:3], t.shape[3] + 5, dtype=t.dtype, device="cuda")
        wide[..., 3:-2] = t.detach()
        return leaf(wide[..., 3:-2])
    same(odd(q), odd(k), odd(v), odd(do).detach())
    columns = lambda t: leaf(t.detach().transpose(1, 3).contiguous().transpose(1, 3))
    same(columns(q), columns(k), columns(v), columns(do).detach())
    same(q, k, v, do, L.long() + torch.tensor([2 ** 40, 0], device="cuda"))
    same(q, k, v, do, L, torch.stack((mask, ~mask), 2)[:, :, 0])
    same(q, k, v, do, torch.stack((L, L), 1)[:, 0], mask.t().contiguous().t())
    none = cross_attention(q, k, v, L - 1000, mask)
    assert float(none.abs().sum()) == 0
    shared = k.detach()[:1].expand(b, sk, hkv, d)                         # one encoder's states for the whole batch
    assert torch.equal(cross_attention(q, shared, shared), cross_attention(q, shared.contiguous(), shared.contiguous()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        o2 = cross_attention(q, k, v, L, mask)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(o2, want[0])


def test_nothing_to_do_and_partial_gradients():
    from rt_pose_amd.attention import cross_attention
    q, k, v, do, _, _ = case(2, 9, 20, 4, 2, 32, torch.bfloat16, seed=9)
    for a, c in ((q[:, :0], k), (q[:0], k[:0]), (q, k[:, :0])):
        a, c = a.detach().requires_grad_(True), c.detach().requires_grad_(True)
        o = cross_attention(a, c, c)
        assert o.shape == a.shape and float(o.abs().sum()) == 0
        ga, gc = torch.autograd.grad(o, (a, c), torch.ones_like(o))
        assert ga.shape == a.shape and gc.shape == c.shape and float(ga.abs().sum()) + float(gc.abs().sum()) == 0
    o = cross_attention(q, k, v)
    full = torch.autograd.grad(o, (q, k, v), do)
    (gq,) = torch.autograd.grad(cross_attention(q, k.detach(), v.detach()), q, do)
    (gv,) = torch.autograd.grad(cross_attention(q.detach(), k.detach(), v), v, do)
    (gk,) = torch.autograd.grad(cross_attention(q.detach(), k, v.detach()), k, do)
    assert torch.equal(gq, full[0]) and torch.equal(gk, full[1]) and torch.equal(gv, full[2])
    (both,) = torch.autograd.grad(cross_attention(q, k, k), k, do)        # the same tensor as keys and values: the gradients add
    parts = torch.autograd.grad(cross_attention(q, k, k.detach().requires_grad_(True)), k, do)[0]
    z = k.detach().clone().requires_grad_(True)
    (pv,) = torch.autograd.grad(cross_attention(q.detach(), k.detach(), z), z, do)
    assert torch.equal(both, parts + pv)


def test_gradients_against_differences():
    from rt_pose_amd.attention import cross_attention
    q, k, v, do, lens, mask = case(1, 3, 20, 2, 1, 8, torch.float16, [17], 0.8, seed=21)
    seen = seen_of(1, 20, lens, mask)
    o = cross_attention(q, k, v, lens.cuda(), mask)
    grads = torch.autograd.grad(o, (q, k, v), do)
    bounds = reference(q, k, v, seen, 8 ** -0.5, do)[1:]
    f = lambda a, b, c: float((reference64(a, b, c, seen) * do.double()).sum())

    def reference64(a, b, c, seen):
        h = lambda x: x.transpose(1, 2)
        s = (h(a) @ h(b).transpose(2, 3).repeat_interleave(2, 1) * 8 ** -0.5).masked_fill(~seen[:, None, None, :], float("-inf"))
        return h(torch.softmax(s, 3) @ h(c).repeat_interleave(2, 1))
    step = 1e-5
    for i, (g, (_, tol)) in enumerate(zip(grads, bounds)):
        for at in range(0, g.numel(), 7):
            x = [t.detach().double().clone() for t in (q, k, v)]
            x[i].view(-1)[at] += step
            up = f(*x)
            x[i].view(-1)[at] -= 2 * step
            num = (up - f(*x)) / (2 * step)               # central differences in 64 bits: off by about step^2 and 1e-16 / step
            assert abs(float(g.reshape(-1)[at]) - num) <= float(tol.reshape(-1)[at]) + 1e-8


def test_captured_and_replayed():
    from rt_pose_amd.attention import cross_attention
    q, k, v, do, lens, mask = case(2, 20, 900, 4, 2, 64, torch.bfloat16, [900, 500], 0.9, seed=13)
    L = lens.cuda()

    def step():
        o = cross_attention(q, k, v, L, mask)
        return (o, *torch.autograd.grad(o, (q, k, v), do))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):                                    # two graphs: each has its own workspace
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, out))
    for seed in range(30, 33):
        with torch.no_grad():
            q.copy_(rnd(2, 20, 4, 64, seed=seed, dtype=torch.bfloat16))
            L.copy_(torch.tensor([900 - seed, 10 * seed]))
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        want = [t.detach().clone() for t in step()]
        for _, out in graphs:
            assert all(torch.equal(a, c) for a, c in zip(out, want))


def test_strides_beyond_what_the_kernels_index_and_sizes_beyond_all():
    from rt_pose_amd.attention import cross_attention
    q, k, v, do, _, _ = case(1, 3, 3, 2, 1, 8, torch.bfloat16, seed=40)
    o = cross_attention(q, k, v)
    want = (o, *torch.autograd.grad(o, (q, k, v), do))

    def far(t, ss):                                                       # tokens `ss` elements apart
        big = torch.zeros(2 * ss + t[0, 0].numel(), dtype=t.dtype, device="cuda")
        view = big.as_strided(t.shape, (0, ss, 8, 1))
        view.copy_(t.detach())
        return view
    for ss in (2 ** 23, 2 ** 23 + 8):
        q2, k2, v2 = (far(t, ss).requires_grad_(True) for t in (q, k, v))
        o2 = cross_attention(q2, k2, v2)
        got = (o2, *torch.autograd.grad(o2, (q2, k2, v2), far(do, ss)))
        assert all(torch.equal(a, c) for a, c in zip(got, want))
    line = torch.zeros(8, dtype=torch.bfloat16, device="cuda")
    for sq, sk, hq in ((2 ** 32 + 1, 1, 1), (1, 2 ** 32 + 1, 1), (1, 1, 2 ** 32 + 1)):
        with pytest.raises(ValueError):
            cross_attention(line.expand(1, sq, hq, 8), line.expand(1, sk, 1, 8), line.expand(1, sk, 1, 8))


def test_saved_operands_that_come_back_elsewhere_or_in_another_layout():
    from rt_pose_amd.attention import cross_attention
    q, k, v, do, lens, mask = case(2, 20, 150, 4, 2, 32, torch.float16, [150, 70], 0.8, seed=50)
    L = lens.cuda()
    want = torch.autograd.grad(cross_attention(q, k, v, L, mask), (q, k, v), do)
    with torch.autograd.graph.save_on_cpu():
        o = cross_attention(q, k, v, L, mask)
    assert all(torch.equal(a, c) for a, c in zip(torch.autograd.grad(o, (q, k, v), do), want))
    # back at the same address, but packed: the place of q is the front of a wider tensor's
    wide = torch.zeros(2, 20, 8, 32, dtype=q.dtype, device="cuda")
    q2 = wide[:, :, ::2]
    q2.copy_(q.detach())
    q2 = q2.detach().requires_grad_(True)

    def back(t):
        if t[0] != wide.data_ptr():
            return t[1]
        packed = wide.view(-1)[:t[1].numel()].view(t[1].shape)
        packed.copy_(t[1])
        return packed
    with torch.autograd.graph.saved_tensors_hooks(lambda t: (t.data_ptr(), t.detach().clone(memory_format=torch.contiguous_format)), back):
        o = cross_attention(q2, k, v, L, mask)
    assert all(torch.equal(a, c) for a, c in zip(torch.autograd.grad(o, (q2, k, v), do), want))


def test_two_calls_at_once():
    from rt_pose_amd.attention import cross_attention
    cases = [case(2, 1, 3000, 8, 2, 64, torch.bfloat16, [3000, 1700], 0.9, seed=60), case(2, 200, 700, 4, 4, 64, torch.bfloat16, [700, 9], 0.9, seed=70)]

    def step(c):
        q, k, v, do, lens, mask = c
        o = cross_attention(q, k, v, lens.to("cuda", non_blocking=True), mask)
        return (o, *torch.autograd.grad(o, (q, k, v), do))
    want = [step(c) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = []
    for _ in range(3):
        for c, s in zip(cases, streams):
            with torch.cuda.stream(s):
                got.append(step(c))
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(g, want[i % 2]))


@pytest.mark.parametrize("b,sk,hkv,d", [(2, 4000, 1, 128), (7, 1500, 8, 16), (8, 2560, 2, 64), (33, 900, 1, 32), (64, 700, 2, 8), (64, 600, 8, 32), (65, 600, 1, 96)])
def test_lengths_of_every_kind(b, sk, hkv, d):
    """Few rows: runs of keys follow the entries' lengths, from none at all to every entry full."""
    from rt_pose_amd.attention import cross_attention
    g = torch.Generator().manual_seed(b)
    kinds = [torch.zeros(b), torch.full((b,), sk), torch.rand(b, generator=g) * (sk + 1), (torch.rand(b, generator=g) < 0.3) * sk, torch.arange(b), torch.ones(b)]
    kinds[3][b // 2] = sk
    q, k, v, do, _, mask = case(b, 2, sk, 2 * hkv, hkv, d, torch.bfloat16, None, 0.8, seed=b)
    for i, kind in enumerate(kinds):
        lens = kind.int()
        m = mask if i % 2 else None
        o = cross_attention(q, k, v, lens.cuda(), m)
        got = (o, *torch.autograd.grad(o, (q, k, v), do))
        check(got, reference(q, k, v, seen_of(b, sk, lens, m), d ** -0.5, do))
