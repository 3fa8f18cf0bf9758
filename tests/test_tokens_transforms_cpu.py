"""The token operators under forward mode and under a trace, without a GPU: the Python layer as it is, with the native call replaced by one that
notes its name and fills the output."""
import ctypes as C

import pytest
import torch
import torch.autograd.forward_ad as fw

pytestmark = pytest.mark.filterwarnings("ignore")      # a trace warns of every size that it turns into a number


@pytest.fixture
def native(monkeypatch):
    """The native calls made; each fills its first output with the byte 0x40."""
    from rt_pose_amd import _lib, attention, fp8, rmsnorm
    made = []
    entries = {"rtp_xattn_forward": lambda a, o, *_: (o, a._obj.b * a._obj.sq * a._obj.hq * a._obj.d * 2),
               "rtp_quantize_fp8": lambda x, x_rs, turned, q, q_rs, scale, rows, *_: (q, rows * q_rs),
               "rtp_matmul_fp8": lambda a, lda, sa, b, ldb, sb, square, out, m, n, k, t: (out, m * n * (4 if t == 0 else 2)),
               "rtp_rmsnorm_forward": lambda x, x_rs, r, r_rs, w, wt, y, s, rows, h, t, eps: (y, rows * h * (4 if t == 0 else 2)),
               "rtp_rmsnorm_fp8_forward": lambda x, x_rs, r, r_rs, w, wt, q, q_rs, scale, s, rows, *_: (q, rows * q_rs)}

    def call(name, t, *args):
        made.append(name)
        fn = C.CFUNCTYPE(C.c_int, *_lib.PROTOTYPES[name][:-1])(lambda *a: 0)      # takes what the native entry takes
        fn(*args)
        at, n = entries[name](*args)
        if n:
            C.memset(at, 0x40, n)

    for module in (attention, fp8, rmsnorm):
        monkeypatch.setattr(module, "same_device", lambda *a: None)
        monkeypatch.setattr(module, "call", call)
    return made


def filled(t):
    return bool((t.contiguous().view(torch.uint8) == 0x40).all())


def traced(f, *args):
    with torch.no_grad():
        return torch.jit.trace(f, args, check_trace=False)


def tangents_are_refused(f, *tensors):
    for i in range(len(tensors)):
        with fw.dual_level():
            args = list(tensors)
            args[i] = fw.make_dual(args[i], torch.ones_like(args[i]))
            with pytest.raises(NotImplementedError):
                f(*args)


def qkv(b=2, sq=3, sk=5):
    return [torch.zeros(b, n, h, 16, dtype=torch.bfloat16) for n, h in ((sq, 4), (sk, 2), (sk, 2))]


def test_cross_attention_refuses_tangents(native):
    from rt_pose_amd.attention import cross_attention
    tangents_are_refused(cross_attention, *qkv())


def test_cross_attention_is_a_node_of_a_trace(native):
    from rt_pose_amd.attention import cross_attention
    lens = torch.tensor([5, 2])
    f = traced(lambda q, k, v, n: cross_attention(q, k, v, key_lens=n), *qkv(), lens)
    assert "CrossAttentionFunction" in str(f.graph)
    del native[:]
    q, k, v = qkv(2, 7, 9)
    out = f(q, k, v, lens)                                         # other sizes than the traced ones
    assert native == ["rtp_xattn_forward"] and out.shape == q.shape and filled(out)
    assert filled(f(q.transpose(1, 2).contiguous().transpose(1, 2), k, v, lens))      # another layout
    with pytest.raises(Exception, match="expected"):               # checked at every call: nothing is read that is not there
        f(q, k, v[:, :4], lens)
    assert f(q.requires_grad_(True), k, v, lens).requires_grad


def test_cross_attention_keeps_nothing_where_no_gradient_is_asked_for(native):
    from rt_pose_amd.attention import cross_attention
    q, k, v = qkv()
    assert not cross_attention(q, k, v).requires_grad
    q.requires_grad_(True)
    with torch.no_grad():
        assert not cross_attention(q, k, v).requires_grad
    o = cross_attention(q, k, v)
    assert o.requires_grad and o.grad_fn.saved_tensors[0].data_ptr() == q.data_ptr()


def eight(rows, cols, square):
    return torch.zeros(rows, cols).to(torch.float8_e4m3fn), torch.ones(-(-rows // 128) if square else rows, -(-cols // 128))


def test_the_8_bit_entries_refuse_tangents(native):
    from rt_pose_amd.fp8 import matmul_fp8, quantize_fp8
    from rt_pose_amd.rmsnorm import add_rms_norm_fp8
    x, w = torch.ones(3, 40, dtype=torch.bfloat16), torch.ones(40)
    tangents_are_refused(quantize_fp8, x)
    tangents_are_refused(add_rms_norm_fp8, x, x, w)
    tangents_are_refused(lambda x, w: add_rms_norm_fp8(x, None, w), x, w)
    (a, sa), (b, sb) = eight(3, 40, False), eight(5, 40, True)
    tangents_are_refused(lambda sa, sb: matmul_fp8(a, sa, b, sb), sa, sb)


def test_the_8_bit_entries_carry_no_gradient(native):
    from rt_pose_amd.fp8 import matmul_fp8, quantize_fp8
    from rt_pose_amd.rmsnorm import add_rms_norm_fp8
    x, w = torch.ones(3, 40, requires_grad=True), torch.ones(40, requires_grad=True)
    (a, sa), (b, sb) = eight(3, 40, False), eight(5, 40, True)
    outs = [*quantize_fp8(x), *add_rms_norm_fp8(x, x, w), *add_rms_norm_fp8(x, None, w)[:2], matmul_fp8(a, sa.requires_grad_(True), b, sb),
            matmul_fp8(a[:0], sa[:0], b, sb)]
    assert not any(t.requires_grad for t in outs) and add_rms_norm_fp8(x, None, w)[2] is x
    for t in outs:
        t.copy_(torch.zeros_like(t))                               # the caller's own, to overwrite as well


def test_the_8_bit_entries_are_nodes_of_a_trace(native):
    from rt_pose_amd.fp8 import matmul_fp8, quantize_fp8
    from rt_pose_amd.rmsnorm import add_rms_norm_fp8
    x, w = torch.ones(3, 40), torch.ones(40)
    f = traced(lambda x: quantize_fp8(x, (128, 128)), x)
    q, scale = f(torch.ones(150, 300))
    assert native[-1] == "rtp_quantize_fp8" and q.shape == (150, 300) and scale.shape == (2, 3) and filled(q)
    f = traced(add_rms_norm_fp8, x, x, w)
    q, scale, s = f(torch.ones(2, 7, 40), torch.ones(2, 7, 40), w)
    assert native[-1] == "rtp_rmsnorm_fp8_forward" and q.shape == s.shape == (2, 7, 40) and scale.shape == (2, 7, 1) and filled(q)
    with pytest.raises(Exception, match="expected"):               # rows that the weight does not have
        f(torch.ones(3, 41), torch.ones(3, 41), w)
    f = traced(lambda x, w: add_rms_norm_fp8(x, None, w), x, w)
    z = torch.ones(5, 40)
    q, scale, s = f(z, w)
    assert q.shape == (5, 40) and filled(q) and torch.equal(s, z)
    (a, sa), (b, sb) = eight(3, 40, False), eight(5, 40, True)
    f = traced(lambda a, sa, b, sb: matmul_fp8(a, sa, b, sb, torch.float16), a, sa, b, sb)
    (a, sa), (b, sb) = eight(4, 300, False), eight(200, 300, True)
    out = f(a, sa, b, sb)
    assert native[-1] == "rtp_matmul_fp8" and out.shape == (4, 200) and out.dtype == torch.float16 and filled(out)
    with pytest.raises(Exception, match="expected"):
        f(a, sa[:3], b, sb)


def test_the_norms_refuse_tangents(native):
    from rt_pose_amd.rmsnorm import add_rms_norm, rms_norm
    x, w = torch.ones(3, 40, dtype=torch.bfloat16), torch.ones(40)
    tangents_are_refused(rms_norm, x, w)
    tangents_are_refused(add_rms_norm, x, x, w)


def test_the_norms_check_at_every_call_of_a_trace(native):
    from rt_pose_amd.rmsnorm import RMSNorm, add_rms_norm, rms_norm
    x, w = torch.ones(3, 40), torch.ones(40)
    f, g, m = traced(rms_norm, x, w), traced(add_rms_norm, x, x, w), traced(RMSNorm(40), x)
    z = torch.ones(2, 7, 40)
    assert filled(f(z, w)) and filled(g(z, z, w)[0]) and filled(m(z))
    wide = torch.ones(3, 41)
    for call in (lambda: f(wide, w), lambda: g(wide, wide, w), lambda: g(x, wide, w), lambda: m(wide)):
        done = len(native)
        with pytest.raises(Exception, match="rms norm"):
            call()
        assert len(native) == done                                 # nothing is read that is not there


def test_a_weight_that_is_not_trained_costs_no_gradient(monkeypatch):
    """Neither the weight's gradient nor its partial rows are asked for."""
    from rt_pose_amd import rmsnorm
    made = []
    monkeypatch.setattr(rmsnorm, "same_device", lambda *a: None)
    monkeypatch.setattr(rmsnorm, "call", lambda name, t, *args: made.append((name, args)))
    for trained in (False, True):
        x, w = torch.ones(3, 40, requires_grad=True), torch.ones(40, requires_grad=trained)
        for f in (lambda: rmsnorm.rms_norm(x, w), lambda: rmsnorm.add_rms_norm(x, x, w)[0]):
            f().sum().backward()
            name, args = made[-1]
            assert name == "rtp_rmsnorm_backward" and (args[9] is not None) == (args[10] is not None) == trained


def test_a_graph_of_torch_operators_is_refused(monkeypatch):
    """make_fx runs on real tensors and records torch's operators alone: its graph would return an output that nothing has written."""
    from torch.fx.experimental.proxy_tensor import make_fx
    from torch.utils.flop_counter import FlopCounterMode

    from rt_pose_amd import _lib, _tokens, attention, fp8, rmsnorm
    for module in (attention, fp8, rmsnorm):
        monkeypatch.setattr(module, "same_device", lambda *a: None)
    x, w, (q, k, v) = torch.ones(3, 40), torch.ones(40), qkv()
    (a, sa), (b, sb) = eight(3, 48, False), eight(5, 48, True)
    for f, args in ((rmsnorm.rms_norm, (x, w)), (rmsnorm.add_rms_norm, (x, x, w)), (rmsnorm.add_rms_norm_fp8, (x, x, w)), (fp8.quantize_fp8, (x,)),
                    (lambda sa, sb: fp8.matmul_fp8(a, sa, b, sb), (sa, sb)), (attention.cross_attention, (q, k, v))):
        with pytest.raises(NotImplementedError, match="make_fx"):
            make_fx(lambda *t: f(*t))(*args)
    made = []
    monkeypatch.setattr(_tokens, "_current_device", lambda: -1)
    monkeypatch.setattr(_tokens, "_raw_stream", lambda index: None)
    monkeypatch.setattr(_lib, "load", lambda: type("Lib", (), {"rtp_rmsnorm_forward": staticmethod(lambda *a: made.append(1) or 0)}))
    with FlopCounterMode(display=False):                           # other modes only look on
        rmsnorm.rms_norm(x, w)
    assert made


def test_tangents_of_the_gradients_are_refused(monkeypatch):
    """Forward mode over a backward pass: the gradients' derivatives would be lost as the values' would be in the forward pass."""
    from rt_pose_amd import attention, rmsnorm
    made = []
    for module in (attention, rmsnorm):
        monkeypatch.setattr(module, "same_device", lambda *a: None)
        monkeypatch.setattr(module, "call", lambda name, *a: made.append(name))
    x, w, (q, k, v) = torch.ones(3, 40, requires_grad=True), torch.ones(40), qkv()
    q.requires_grad_(True)
    for f, t in ((lambda: rmsnorm.rms_norm(x, w), x), (lambda: rmsnorm.add_rms_norm(x, x.detach(), w)[0], x), (lambda: rmsnorm.add_rms_norm(x, x.detach(), w)[1], x),
                 (lambda: attention.cross_attention(q, k, v), q)):
        with fw.dual_level():
            y = f()
            one = torch.ones_like(y)
            with pytest.raises(NotImplementedError):
                torch.autograd.grad(y, t, fw.make_dual(one, one))
            y = f()
            torch.autograd.grad(y, t, one)                         # a level alone is no tangent
