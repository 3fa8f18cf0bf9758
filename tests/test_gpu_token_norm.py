"""RMS norm with the residual's addition, its 8-bit form and quantising against plain 64-bit implementations.

Tolerances: one rounding to the output's type is half a step, finfo(t).eps / 2 of the value; sums of n fp32 terms are off by at most
(about 40 + n / 1024) roundings of 2^-24 of the sum of magnitudes (each lane adds <= 64 terms in a row, trees join the lanes, partial rows
are added in blocks): U below, elementwise on the magnitudes that enter."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 64 * 2.0 ** -24
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def rnd(*shape, seed, dtype, scale=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype).cuda()


def half(t):
    return torch.finfo(t).eps / 2


def close(got, want, tol, what):
    # below its smallest normal 2^-14 an fp16 value has steps of 2^-24, whatever its size: a rounding there is off by up to 2^-25, which half a
    # step RELATIVE to the value does not cover (fp32 and bf16: 2^-150 and 2^-134, never reached by these inputs)
    got, want = got.detach(), want.detach()
    bad = (got.double() - want).abs() - tol.detach() - (2.0 ** -25 if got.dtype == torch.float16 else 0.0)
    assert got.shape == want.shape and bool((bad <= 0).all()), "%s: over its bound by %g" % (what, float(bad.max()))


def norm64(s, w, eps):
    s, w = s.double(), w.double()
    return s / torch.sqrt((s * s).mean(-1, keepdim=True) + eps) * w


ROWS = [(1, 1), (3, 7), (5, 128), (130, 129), (7, 512), (33, 777), (9, 1024), (4, 1999), (3, 4096), (2, 5001), (2, 8192), (2, 16001)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,h", ROWS)
@pytest.mark.parametrize("w32", [False, True])
def test_forward_backward(rows, h, dtype, w32):
    from rt_pose_amd.rmsnorm import add_rms_norm
    eps = 1e-5
    x, r = rnd(rows, h, seed=1, dtype=dtype).requires_grad_(True), rnd(rows, h, seed=2, dtype=dtype, scale=3.0).requires_grad_(True)
    w = (1 + rnd(h, seed=3, dtype=torch.float32, scale=0.3)).to(torch.float32 if w32 else dtype).requires_grad_(True)
    dy, ds = rnd(rows, h, seed=4, dtype=dtype), rnd(rows, h, seed=5, dtype=dtype)
    y, s = add_rms_norm(x, r, w, eps)
    want_s = (x.double() + r.double()).to(dtype)      # two values of one type: their exact sum fits fp32 wherever it is not just the larger one
    assert torch.equal(s, want_s) and y.dtype == dtype
    y64 = norm64(want_s, w, eps)
    close(y, y64, y64.abs() * (half(dtype) + U), "y")
    dx, dr, dw = torch.autograd.grad((y, s), (x, r, w), (dy, ds))
    assert torch.equal(dx, dr) and dw.dtype == w.dtype
    s64, w64 = want_s.double(), w.double().detach()
    root = torch.sqrt((s64 * s64).mean(-1, keepdim=True) + eps)
    g, xh = dy.double() * w64, s64 / root
    own = (g - xh * (g * xh).mean(-1, keepdim=True)) / root
    mag = (g.abs() + xh.abs() * (g * xh).abs().mean(-1, keepdim=True)) / root + ds.double().abs()
    close(dx, own + ds.double(), (own + ds.double()).abs() * half(dtype) + U * mag, "dx")
    dw64, dwm = (dy.double() * xh).sum(0), (dy.double() * xh).abs().sum(0)
    close(dw, dw64, dw64.abs() * half(w.dtype) + U * dwm, "dw")


def test_gradients_against_differences():
    from rt_pose_amd.rmsnorm import add_rms_norm
    x, r, w = (rnd(*s, seed=i, dtype=torch.float32) for i, s in enumerate([(3, 40), (3, 40), (40,)]))
    dy, ds = rnd(3, 40, seed=7, dtype=torch.float32).double(), rnd(3, 40, seed=8, dtype=torch.float32).double()
    leaves = [t.clone().requires_grad_(True) for t in (x, r, w)]
    y, s = add_rms_norm(*leaves, 1e-5)
    grads = torch.autograd.grad((y, s), leaves, (dy.float(), ds.float()))
    f = lambda a, b, c: (norm64(a + b, c, 1e-5) * dy).sum() + ((a + b) * ds).sum()
    step = 1e-5
    for i, (t, g) in enumerate(zip((x, r, w), grads)):
        for k in (0, t.numel() // 2, t.numel() - 1):
            at = [v.double().clone() for v in (x, r, w)]
            at[i].view(-1)[k] += step
            up = f(*at)
            at[i].view(-1)[k] -= 2 * step
            # central difference in 64 bits: truncation ~ step^2, rounding ~ 1e-16 * |f| / step; the gradient's own bound is far wider
            num = float((up - f(*at)) / (2 * step))
            assert abs(float(g.view(-1)[k]) - num) < 2e-4 * max(1.0, abs(num))


@pytest.mark.parametrize("dtype", TYPES)
def test_without_residual_and_only_one_output_used(dtype):
    from rt_pose_amd.rmsnorm import RMSNorm, add_rms_norm, rms_norm
    x = rnd(2, 5, 96, seed=1, dtype=dtype).requires_grad_(True)
    w = rnd(96, seed=2, dtype=torch.float32)
    y64 = norm64(x, w, 1e-6)
    close(rms_norm(x, w), y64, y64.abs() * (half(dtype) + U), "y")
    r = rnd(2, 5, 96, seed=3, dtype=dtype)
    y, s = add_rms_norm(x, r, w)
    (only_stream,) = torch.autograd.grad(s.float().sum(), x, retain_graph=True)
    assert torch.equal(only_stream, torch.ones_like(x))
    (only_y,) = torch.autograd.grad(y, x, torch.ones_like(y))
    z = s.detach().requires_grad_(True)
    (alone,) = torch.autograd.grad(rms_norm(z, w), z, torch.ones_like(y))
    assert torch.equal(only_y, alone)
    m = RMSNorm(96).cuda()
    assert torch.equal(m(x.detach()), rms_norm(x.detach(), torch.ones(96, device="cuda")))
    assert torch.equal(m(x.detach(), r)[1], s.detach())


@pytest.mark.parametrize("h", [64, 333, 1024, 4100])
def test_strides_and_streams(h):
    from rt_pose_amd.rmsnorm import add_rms_norm, add_rms_norm_fp8
    wide = rnd(6, 2 * h + 3, seed=1, dtype=torch.bfloat16)
    x, r = wide[:, 1:1 + h], wide[:, h + 2:2 * h + 2].flip(0)
    w = rnd(2 * h, seed=2, dtype=torch.float32)[::2]
    got, want = add_rms_norm(x, r, w), add_rms_norm(x.contiguous(), r.contiguous(), w.contiguous())
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    row = r[:1].expand(6, h)                              # one residual for all rows: stride 0
    assert torch.equal(add_rms_norm(x, row, w)[0], add_rms_norm(x, row.contiguous(), w)[0])
    assert torch.equal(add_rms_norm(x.t().contiguous().t(), r, w)[0], want[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        q, sc, s = add_rms_norm_fp8(x, r, w)
    torch.cuda.current_stream().wait_stream(side)
    q2, sc2, s2 = add_rms_norm_fp8(x, r, w)
    assert torch.equal(q.float(), q2.float()) and torch.equal(sc, sc2) and torch.equal(s, s2)


def test_backward_is_the_same_every_time_and_takes_any_gradient_strides():
    from rt_pose_amd.rmsnorm import rms_norm
    x, w = rnd(3000, 200, seed=1, dtype=torch.bfloat16).requires_grad_(True), rnd(200, seed=2, dtype=torch.bfloat16).requires_grad_(True)
    dy = rnd(3000, 200, seed=3, dtype=torch.bfloat16)
    runs = [torch.autograd.grad(rms_norm(x, w), (x, w), g) for g in (dy, dy, dy.t().contiguous().t())]
    for other in runs[1:]:
        assert torch.equal(runs[0][0], other[0]) and torch.equal(runs[0][1], other[1])
    one = torch.autograd.grad(rms_norm(x, w).float().sum(), (x, w))     # a gradient broadcast from one value
    full = torch.autograd.grad(rms_norm(x, w), (x, w), torch.ones_like(x))
    assert torch.equal(one[0], full[0]) and torch.equal(one[1], full[1])


def test_no_rows_and_rows_without_finite_values():
    from rt_pose_amd.rmsnorm import add_rms_norm, add_rms_norm_fp8, rms_norm
    x = torch.empty(0, 64, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    w = torch.ones(64, device="cuda", requires_grad=True)
    y, s = add_rms_norm(x, x, w)
    gx, gw = torch.autograd.grad((y, s), (x, w), (y, s))
    assert y.shape == (0, 64) and gx.shape == (0, 64) and float(gw.abs().sum()) == 0
    q, sc, s = add_rms_norm_fp8(x, None, w)
    assert q.shape == (0, 64) and sc.shape == (0, 1) and s is x
    z = torch.zeros(3, 64, device="cuda")
    z[1, 5], z[2, 7] = float("nan"), float("inf")
    y = rms_norm(z, torch.ones(64, device="cuda"))
    assert float(y[0].abs().sum()) == 0 and bool(y[1].isnan().all()) and bool(y[2, 7].isnan()) and float(y[2, :7].abs().sum()) == 0


def quant64(x, square):
    """q and scale by the rule, on the CPU: the maximum is exact, 448 / a and x * up are single fp32 roundings."""
    x = x.float().cpu()
    rows, cols = x.shape
    kb, rb = -(-cols // 128), -(-rows // 128)
    full = torch.zeros(rb * 128, kb * 128)
    full[:rows, :cols] = x.nan_to_num(nan=0.0, posinf=float("inf"), neginf=float("-inf")).abs()
    a = full.view(rb, 128, kb, 128).amax((1, 3)) if square else full.view(rb * 128, kb, 128).amax(2)[:rows]
    a = a.clamp_min(2.0 ** -100)
    up = torch.tensor(448.0) / a
    wide = up.repeat_interleave(128, 1)[:, :cols]
    wide = wide.repeat_interleave(128, 0)[:rows] if square else wide
    return (x * wide).to(torch.float8_e4m3fn), a / 448.0


QUANT = [(1, 1), (1, 300), (5, 128), (130, 129), (257, 77), (128, 640), (3, 2050)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", QUANT)
@pytest.mark.parametrize("square", [False, True])
@pytest.mark.parametrize("turned", [False, True])
def test_quantize(rows, cols, square, turned, dtype):
    from rt_pose_amd.fp8 import quantize_fp8
    x = rnd(rows, cols, seed=rows, dtype=torch.float32) * torch.logspace(-6, 3, cols).cuda()
    x = x.to(dtype)
    x[0, cols // 2] = 0
    x = x.t().contiguous().t() if turned else x
    q, scale = quantize_fp8(x, (128, 128) if square else (1, 128))
    wq, ws = quant64(x, square)
    assert q.shape == x.shape and scale.shape == ws.shape and q.stride(0) % 16 == 0
    assert torch.equal(scale.cpu(), ws)
    assert torch.equal(q.cpu().view(torch.uint8), wq.view(torch.uint8))


@pytest.mark.parametrize("turned", [False, True])
@pytest.mark.parametrize("square", [False, True])
def test_quantize_special_values(square, turned):
    from rt_pose_amd.fp8 import quantize_fp8
    x = torch.zeros(256, 384, device="cuda")
    x[0, 3], x[0, 4] = float("nan"), 5.0          # NaN stays alone, the scale is the others'
    x[1, 130], x[1, 131] = float("-inf"), 1.0     # the whole block reads back as NaN
    x[130, 0] = 1e-38                             # below the floor: zero, not a division by zero
    x[131, 1] = 3e38                              # near the type's end
    x = x.t().contiguous().t() if turned else x
    q, scale = quantize_fp8(x, (128, 128) if square else (1, 128))
    up = (lambda r, c: scale[r // 128, c // 128]) if square else (lambda r, c: scale[r, c // 128])
    val = lambda r, c: float(q[r, c].float() * up(r, c))
    assert val(0, 3) != val(0, 3) and val(0, 4) == pytest.approx(5.0, rel=1e-6)
    assert val(1, 130) != val(1, 130) and val(1, 131) != val(1, 131)
    assert val(131, 1) == pytest.approx(3e38, rel=1e-6) and val(130, 0) == 0.0
    assert bool(torch.isfinite(q[200].float()).all()) and float(q[200].float().abs().sum()) == 0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,h", ROWS)
@pytest.mark.parametrize("residual", [False, True])
def test_norm_fp8(rows, h, residual, dtype):
    from rt_pose_amd.rmsnorm import add_rms_norm_fp8
    x, r = rnd(rows, h, seed=1, dtype=dtype), rnd(rows, h, seed=2, dtype=dtype)
    w = 1 + rnd(h, seed=3, dtype=torch.float32, scale=0.3)
    q, scale, s = add_rms_norm_fp8(x, r if residual else None, w, 1e-5)
    want_s = (x.double() + r.double()).to(dtype) if residual else x
    assert torch.equal(s, want_s) and q.dtype == torch.float8_e4m3fn and q.shape == x.shape
    y = norm64(want_s, w, 1e-5)
    kb = -(-h // 128)
    a = torch.nn.functional.pad(y.abs(), (0, kb * 128 - h)).view(rows, kb, 128).amax(2).clamp_min(2.0 ** -100)
    close(scale, a / 448, a / 448 * U, "scale")
    wide = scale.double().repeat_interleave(128, 1)[:, :h]
    # e4m3: half a step of 2^-3 relative, or of its smallest step 2^-9 below 2^-6; the value rounded is off by U
    close(q.double() * wide, y, torch.maximum(y.abs() * 2.0 ** -4, wide * 2.0 ** -10) * (1 + U) + y.abs() * U, "q * scale")
    assert bool((q.float().abs().amax(1) >= 448 * (1 - U)).any())


def test_captured_and_replayed():
    from rt_pose_amd.rmsnorm import add_rms_norm, add_rms_norm_fp8
    x, r = rnd(300, 640, seed=1, dtype=torch.bfloat16).requires_grad_(True), rnd(300, 640, seed=2, dtype=torch.bfloat16)
    w, dy = rnd(640, seed=3, dtype=torch.float32).requires_grad_(True), rnd(300, 640, seed=4, dtype=torch.bfloat16)

    def step():
        y, s = add_rms_norm(x, r, w)
        return (y, s, *torch.autograd.grad((y, s), (x, w), (dy, dy)), *add_rms_norm_fp8(x.detach(), r, w.detach())[:2])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in range(10, 13):
        with torch.no_grad():
            x.copy_(rnd(300, 640, seed=seed, dtype=torch.bfloat16))
        graph.replay()
        torch.cuda.synchronize()
        got = [o.detach().float().clone() for o in out]
        assert all(torch.equal(a, b.detach().float()) for a, b in zip(got, step()))


def test_the_same_rows_twice_broadcast_rows_and_widths_beyond():
    from rt_pose_amd.fp8 import quantize_fp8
    from rt_pose_amd.rmsnorm import RMSNorm, add_rms_norm, add_rms_norm_fp8, rms_norm
    x, w, dy, ds = (rnd(6, 200, seed=80 + i, dtype=torch.float32) for i in range(4))
    x.requires_grad_(True)
    r = x.detach().clone().requires_grad_(True)
    y, s = add_rms_norm(x, x, w[0])                                        # the residual is x itself: both gradients add
    (g,) = torch.autograd.grad((y, s), x, (dy, ds))
    y2, s2 = add_rms_norm(x, r, w[0])
    gx, gr = torch.autograd.grad((y2, s2), (x, r), (dy, ds))
    assert torch.equal(y, y2) and torch.equal(s, s2) and torch.equal(gx, gr) and torch.equal(g, gx + gr)
    x.grad = r.grad = None
    torch.autograd.backward(add_rms_norm(x, r, w[0]), (dy, ds))            # one tensor is the gradient of both: each leaf keeps its own
    x.grad.zero_()
    assert torch.equal(r.grad, gr)
    row = rnd(200, seed=90, dtype=torch.bfloat16)
    many = row.expand(5, 3, 200)
    assert torch.equal(rms_norm(many, row), rms_norm(many.contiguous(), row))
    for a, b in zip(quantize_fp8(row.expand(300, 200), (128, 128)), quantize_fp8(row.repeat(300, 1), (128, 128))):
        assert torch.equal(a.float(), b.float())
    columns = row[:, None].expand(200, 300)                                # a transpose's view whose columns are all the same memory
    for block in ((1, 128), (128, 128)):
        for a, b in zip(quantize_fp8(columns, block), quantize_fp8(columns.contiguous(), block)):
            assert torch.equal(a.float(), b.float())
    wide = torch.zeros(1, 16385, device="cuda")
    for call in (lambda: rms_norm(wide, wide[0]), lambda: add_rms_norm_fp8(wide, None, wide[0]), lambda: RMSNorm(16385).cuda()(wide, wide)):
        with pytest.raises(NotImplementedError):
            call()
    for n in (2 ** 30 + 1, 2 ** 32 + 8):
        with pytest.raises(ValueError):
            quantize_fp8(wide[:, :1].expand(1, n))


@pytest.mark.parametrize("h", [2, 8, 9, 15, 16, 121, 127, 505, 520, 1000, 1023, 1025, 2047, 2056, 4090, 8191, 8200, 12345, 16383])
def test_every_kind_of_width(h):
    """Whole, ragged and short rows at each of the kernels' widths, odd strides and an odd start among them."""
    from rt_pose_amd.fp8 import quantize_fp8
    for dtype in TYPES:
        test_forward_backward(6, h, dtype, dtype != torch.float32)
        test_norm_fp8(5, h, True, dtype)
    for square in (False, True):
        test_quantize(130, h, square, False, torch.bfloat16)
        test_quantize(3, h, square, False, torch.float32)
        wide = rnd(4, h + 3, seed=h, dtype=torch.float16)
        block = (128, 128) if square else (1, 128)
        for a, b in zip(quantize_fp8(wide[:, 1:-2], block), quantize_fp8(wide[:, 1:-2].clone(), block)):
            assert torch.equal(a.float(), b.float())
