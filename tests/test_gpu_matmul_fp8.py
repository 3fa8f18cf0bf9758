"""matmul_fp8 against the 64-bit product of what its operands stand for.

Tolerance, fp32 output: products of two e4m3 values are exact; a block's 128 are added in fp32 (<= 128 roundings of the sum of magnitudes), then
scaled (two roundings) and added to the running sum (one rounding per block): (132 + ceil(k / 128)) 2^-24 of the sum of magnitudes.
bf16 and fp16 output: half a step of the type besides (and for fp16 half of its smallest step), and what the 8-bit matrix instruction leaves out:
it adds groups of eight neighbouring products at 14 bits, so that each of the seven others loses less than 2^-13 of the group's largest --
found with one large product and small ones beside it: 2^16 + 2^(16 - n) keeps the small one up to n = 13 inside the group, up to n = 23 outside."""
import pytest
import torch

pytestmark = pytest.mark.gpu

OUT = [torch.bfloat16, torch.float16, torch.float32]


def operand(rows, cols, square, seed):
    from rt_pose_amd.fp8 import quantize_fp8
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols, generator=g) * torch.exp(torch.randn(rows, 1, generator=g))
    return quantize_fp8(x.cuda(), (128, 128) if square else (1, 128))


def stands_for(q, scale, square):
    s = scale.double().repeat_interleave(128, 1)[:, :q.shape[1]]
    return q.double() * (s.repeat_interleave(128, 0)[:q.shape[0]] if square else s)


def left_out(a, sa, b, sb, square):
    """sum over the groups of eight along k of 7 * 2^-13 * the group's largest product, in what the operands stand for"""
    da, db = stands_for(a, sa, False).abs(), stands_for(b, sb, square).abs()
    total = torch.zeros(a.shape[0], b.shape[0], dtype=torch.float64, device="cuda")
    for k in range(0, a.shape[1], 8):
        top = torch.zeros_like(total)
        for j in range(k, min(k + 8, a.shape[1])):
            top = torch.maximum(top, da[:, j:j + 1] * db[:, j])
        total += top
    return total * (7 * 2.0 ** -13)


def check(out, a, sa, b, sb, square):
    da, db = stands_for(a, sa, False), stands_for(b, sb, square)
    want, mag = da @ db.t(), da.abs() @ db.abs().t()
    tol = (132 + sa.shape[1]) * 2.0 ** -24 * mag
    if out.dtype != torch.float32:
        tol = tol + left_out(a, sa, b, sb, square)
        tol = tol + torch.finfo(out.dtype).eps / 2 * (want.abs() + tol) + (2.0 ** -25 if out.dtype == torch.float16 else 0.0)
    if out.dtype == torch.float16:                  # its largest value is 65504; from 65520 on the nearest value is infinity
        over = want.abs() - tol >= 65520
        assert torch.equal(out[over], torch.copysign(torch.full_like(want, float("inf")), want)[over].half())
        near = over | (want.abs() + tol >= 65520)
        out, want, tol = out.masked_fill(near, 0), want.masked_fill(near, 0), tol
    bad = (out.double() - want).abs() - tol
    assert float(bad.max()) <= 0, float(bad.max())


SIZES = [(1, 1, 1), (1, 16, 128), (4, 130, 1000), (16, 256, 129), (17, 33, 16), (31, 500, 2048), (33, 128, 384), (64, 100, 777), (65, 129, 640),
         (127, 1000, 130), (300, 200, 1030), (1500, 1400, 256), (2000, 1111, 400), (1411, 1600, 127), (4100, 3500, 300), (3584, 4096, 1000),
         (5, 16400, 300), (20, 16400, 1100), (60, 16390, 260), (9, 8200, 520), (30, 8200, 300), (50, 8200, 700), (4000, 4090, 2050)]   # every cut of n, the large tile


@pytest.mark.parametrize("m,n,k", SIZES)
@pytest.mark.parametrize("square", [True, False])
def test_product(m, n, k, square):
    from rt_pose_amd.fp8 import matmul_fp8
    (a, sa), (b, sb) = operand(m, k, False, 1), operand(n, k, square, 2)
    for t in OUT:
        out = matmul_fp8(a, sa, b, sb, out_dtype=t)
        assert out.shape == (m, n) and out.dtype == t
        check(out, a, sa, b, sb, square)


@pytest.mark.parametrize("m,n,k", [(3, 40, 200), (70, 300, 333), (1500, 1300, 520), (4096, 4096, 1049)])
def test_bytes_behind_the_sum_and_other_rows_do_not_count(m, n, k):
    """Operands as views into wider buffers full of NaN bytes, at offsets of 16, with odd strides, and as slices that have to be copied."""
    from rt_pose_amd.fp8 import matmul_fp8
    (a, sa), (b, sb) = operand(m, k, False, 1), operand(n, k, True, 2)
    want = matmul_fp8(a, sa, b, sb)

    def inside(q, lead, ld):
        wide = torch.full((q.shape[0] + 2, ld), 0x7f, dtype=torch.uint8, device="cuda")
        wide[1:-1, lead:lead + q.shape[1]] = q.view(torch.uint8)
        return wide.view(torch.float8_e4m3fn)[1:-1, lead:lead + q.shape[1]]
    up = -(-k // 16) * 16
    for lead, ld in ((16, up + 32), (0, up), (5, up + 48), (3, k + 4)):
        assert torch.equal(matmul_fp8(inside(a, lead, ld), sa, inside(b, lead, ld), sb), want)
    turned = a.view(torch.uint8).t().contiguous().view(torch.float8_e4m3fn).t()
    assert torch.equal(matmul_fp8(turned, sa, b.contiguous(), sb), want)
    last = torch.full((m * k,), 0x7f, dtype=torch.uint8, device="cuda")     # ends with the last value: nothing may be read behind it
    last[:] = a.view(torch.uint8).reshape(-1)
    assert torch.equal(matmul_fp8(last.view(torch.float8_e4m3fn).view(m, k), sa, b, sb), want)
    wide_scale = torch.full((m, 2 * sa.shape[1]), float("nan"), device="cuda")
    wide_scale[:, ::2] = sa
    assert torch.equal(matmul_fp8(a, wide_scale[:, ::2], b, sb), want)


def test_leading_dimensions_empty_operands_and_special_values():
    from rt_pose_amd.fp8 import matmul_fp8
    (a, sa), (b, sb) = operand(6, 200, False, 1), operand(40, 200, True, 2)
    want = matmul_fp8(a, sa, b, sb)
    got = matmul_fp8(a.unflatten(0, (2, 3)), sa.unflatten(0, (2, 3)), b, sb)
    assert got.shape == (2, 3, 40) and torch.equal(got.flatten(0, 1), want)
    assert matmul_fp8(a[:0], sa[:0], b, sb).shape == (0, 40)
    assert matmul_fp8(a, sa, b[:0], sb[:0]).shape == (6, 0)
    a = a.clone()
    a.view(torch.uint8)[2, 7] = 0x7f                                        # NaN: its row, and no other
    got = matmul_fp8(a, sa, b, sb)
    assert bool(got[2].isnan().all()) and torch.equal(got[[0, 1, 3, 4, 5]], want[[0, 1, 3, 4, 5]])


@pytest.mark.parametrize("m", [5, 1500])
def test_scales_of_any_size(m):
    """Scales that overflow or vanish alone but not in their product, and a block whose scale is zero."""
    from rt_pose_amd.fp8 import matmul_fp8
    (a, sa), (b, sb) = operand(m, 300, False, 1), operand(1500, 300, True, 2)
    want = matmul_fp8(a, sa, b, sb, out_dtype=torch.float32)
    big = matmul_fp8(a, sa * 2.0 ** 80, b, sb * 2.0 ** -80, out_dtype=torch.float32)
    assert torch.equal(big, want)
    sa = sa.clone()
    sa[:, 1] = 0
    a = a.clone()
    a[:, 128:256] = 0
    (out,) = (matmul_fp8(a, sa, b, sb, out_dtype=torch.float32),)
    check(out, a, sa, b, sb, True)


def test_the_three_products_of_a_layer():
    """y = x w.T, dx = dy w, dw = dy.T x from operands quantised along their sums: off by the operands' rounding (each value by half a step,
    2^-4, or by half of e4m3's smallest step on its scale), nothing else."""
    from rt_pose_amd.fp8 import matmul_fp8, quantize_fp8
    g = torch.Generator().manual_seed(5)
    x, w, dy = (torch.randn(*s, generator=g).cuda() for s in ((333, 520), (270, 520), (333, 270)))
    for p, q, square in ((x, w, True), (dy, w.t(), True), (dy.t(), x.t(), False)):
        (a, sa), (b, sb) = quantize_fp8(p), quantize_fp8(q, (128, 128) if square else (1, 128))
        out = matmul_fp8(a, sa, b, sb, out_dtype=torch.float32)
        check(out, a, sa, b, sb, square)
        P, Q = p.double(), q.double()
        ea = torch.maximum(P.abs() * 2.0 ** -4, sa.double().repeat_interleave(128, 1)[:, :P.shape[1]] * 2.0 ** -10)
        wide = sb.double().repeat_interleave(128, 1)[:, :Q.shape[1]]
        wide = wide.repeat_interleave(128, 0)[:Q.shape[0]] if square else wide
        eb = torch.maximum(Q.abs() * 2.0 ** -4, wide * 2.0 ** -10)
        bound = (ea @ Q.abs().t() + P.abs() @ eb.t() + ea @ eb.t()) * 1.0001
        assert bool(((out.double() - P @ Q.t()).abs() <= bound).all())


def test_far_rows_and_sizes_beyond():
    from rt_pose_amd.fp8 import matmul_fp8
    (a, sa), (b, sb) = operand(3, 48, False, 90), operand(5, 48, True, 91)
    want = matmul_fp8(a, sa, b, sb)
    for ld in (2 ** 22, 2 ** 22 + 16):                                     # rows further apart than a tile indexes: copied
        far = torch.zeros(4 * ld + 48, dtype=torch.uint8, device="cuda")
        a2, b2 = (far.as_strided((n, 48), (ld, 1)) for n in (3, 5))
        a2.copy_(a.view(torch.uint8))
        assert torch.equal(matmul_fp8(a2.view(a.dtype), sa, b, sb), want)
        assert torch.equal(matmul_fp8(a2[1:2].view(a.dtype), sa[1:2], b, sb), want[1:2])
        b2.copy_(b.view(torch.uint8))
        assert torch.equal(matmul_fp8(a, sa, b2.view(b.dtype), sb), want)
    byte = torch.zeros(1, dtype=torch.uint8, device="cuda").view(a.dtype)
    one = torch.ones(1, device="cuda")
    for m, n, k in ((2 ** 32 + 1, 1, 16), (1, 2 ** 32 + 1, 16), (1, 1, 2 ** 32 + 16), (1, 1, 2 ** 22 + 1)):
        kb = -(-k // 128)
        with pytest.raises(ValueError):
            matmul_fp8(byte.expand(m, k), one.expand(m, kb), byte.expand(n, k), one.expand(n, kb))


@pytest.mark.parametrize("m,n,k", [(4200, 50, 300), (6200, 64, 129), (130, 4200, 390), (1000, 700, 640), (4000, 1000, 130), (520, 1090, 1111)])
@pytest.mark.parametrize("square", [True, False])
def test_tiles_of_half_the_width(m, n, k, square):
    from rt_pose_amd.fp8 import matmul_fp8
    (a, sa), (b, sb) = operand(m, k, False, m + n), operand(n, k, square, m + n + 1)
    for t in OUT:
        check(matmul_fp8(a, sa, b, sb, t), a, sa, b, sb, square)
