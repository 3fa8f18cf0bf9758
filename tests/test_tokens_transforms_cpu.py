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
    from rt_pose_amd import _lib, attention
    made = []
    entries = {"rtp_xattn_forward": lambda a, o, *_: (o, a._obj.b * a._obj.sq * a._obj.hq * a._obj.d * 2)}

    def call(name, t, *args):
        made.append(name)
        fn = C.CFUNCTYPE(C.c_int, *_lib.PROTOTYPES[name][:-1])(lambda *a: 0)      # takes what the native entry takes
        fn(*args)
        at, n = entries[name](*args)
        if n:
            C.memset(at, 0x40, n)

    for module in (attention,):
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
