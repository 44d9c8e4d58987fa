"""Rotary positions, cross attention and root-mean-square norm: what their entry points refuse, checked without a GPU.  The pointers
here are made-up numbers: a call that is not refused fails for want of a device, before anything is launched."""
import ctypes as C
import math

import pytest

import darknet_b200 as dn


def tensor(n, h, w, c, dtype=None, data=0x10000, pitch=None, layout=None):
    return dn.Tensor(data, dn.NHWC if layout is None else layout, dn.BF16 if dtype is None else dtype, n, c, h, w, (c + 7) // 8 * 8 if pitch is None else pitch)


def rope_desc(**kw):
    d = dict(head_dim=64, heads=2, pairs=(8, 12, 12), frames=1, origin=(0, 0, 0), interleaved=0, shared=1, base=10000.0, scale=(1.0, 1.0, 1.0))
    d.update(kw)
    return dn.RopeDesc(d["head_dim"], d["heads"], (C.c_int * 3)(*d["pairs"]), d["frames"], (C.c_int * 3)(*d["origin"]), d["interleaved"], d["shared"], d["base"],
                       (C.c_float * 3)(*d["scale"]))


@pytest.mark.parametrize("kw,word", [
    (dict(head_dim=0), b"heads"), (dict(head_dim=63), b"heads"), (dict(heads=0), b"heads"), (dict(pairs=(0, 0, 0)), b"pairs"),
    (dict(pairs=(-1, 2, 2)), b"pairs"), (dict(pairs=(11, 11, 11)), b"pairs"), (dict(pairs=(1 << 30, 1 << 30, 1 << 30)), b"pairs"), (dict(frames=0), b"frames"),
    (dict(base=0.0), b"base"), (dict(base=-2.0), b"base"), (dict(base=math.nan), b"base"), (dict(base=math.inf), b"base"),
    (dict(scale=(1.0, math.nan, 1.0)), b"scale"), (dict(interleaved=2), b"interleaved"), (dict(shared=-1), b"shared")])
def test_rope_plans_that_are_refused(kw, word):
    L, h = dn.lib(), C.c_void_p(1)
    assert L.dnb_rope_plan_create(C.byref(rope_desc(**kw)), C.byref(h)) == dn.EINVAL
    assert word in L.dnb_last_error() and not h


def test_rope_plan_of_too_many_pairs_is_unsupported():
    L, h = dn.lib(), C.c_void_p()
    assert L.dnb_rope_plan_create(C.byref(rope_desc(head_dim=512, pairs=(0, 100, 100))), C.byref(h)) == dn.EUNSUPPORTED


@pytest.mark.parametrize("x,y,positions", [
    (tensor(1, 4, 4, 120), tensor(1, 4, 4, 120, data=0x20000), None),                       # two heads of 64 do not fit
    (tensor(1, 4, 4, 128), tensor(1, 4, 5, 128, data=0x20000), None),
    (tensor(1, 4, 4, 128), tensor(1, 4, 4, 128, dn.F32, data=0x20000), None),
    (tensor(1, 4, 4, 128), tensor(1, 4, 4, 128, pitch=136), None),                          # in place with another pitch
    (tensor(1, 4, 4, 128, dn.F32, layout=dn.NCHW), tensor(1, 4, 4, 128, dn.F32, data=0x20000, layout=dn.NCHW), None),
    (tensor(1, 4, 4, 128), tensor(1, 4, 4, 128, data=0x20040), None),                       # not 128-byte aligned
    (tensor(1, 4, 4, 128, pitch=132), tensor(1, 4, 4, 128, data=0x20000), None),
    (tensor(1, 4, 4, 128), tensor(1, 4, 4, 128, data=0x20000), 0x30002),                    # positions off their alignment
    (tensor(3, 4, 4, 128), tensor(3, 4, 4, 128, data=0x20000), None)])                      # three images in clips of two frames
def test_rope_calls_that_are_refused(x, y, positions):
    L, h = dn.lib(), C.c_void_p()
    dn.check(L.dnb_rope_plan_create(C.byref(rope_desc(frames=2 if x.n == 3 else 1)), C.byref(h)))
    assert L.dnb_rope_forward(h, C.byref(x), positions, C.byref(y), None) == dn.EINVAL
    assert b"rope" in L.dnb_last_error()
    L.dnb_rope_plan_destroy(h)
    assert L.dnb_rope_forward(None, C.byref(x), positions, C.byref(y), None) == dn.EINVAL


@pytest.mark.parametrize("desc,status", [
    ((8, 3, 64, 0.0), dn.EINVAL), ((0, 1, 64, 0.0), dn.EINVAL), ((8, 0, 64, 0.0), dn.EINVAL), ((8, -8, 64, 0.0), dn.EINVAL), ((8, 8, 60, 0.0), dn.EINVAL),
    ((8, 8, 0, 0.0), dn.EINVAL), ((8, 8, -64, 0.0), dn.EINVAL), ((8, 8, 64, math.nan), dn.EINVAL), ((8, 8, 64, math.inf), dn.EINVAL), ((8, 8, 136, 0.0), dn.EUNSUPPORTED)])
def test_attention_plans_that_are_refused(desc, status):
    L, h = dn.lib(), C.c_void_p(1)
    assert L.dnb_attention_plan_create(C.byref(dn.AttentionDesc(*desc)), C.byref(h)) == status
    assert b"attention" in L.dnb_last_error() and not h
    assert L.dnb_attention_plan_create(None, C.byref(h)) == dn.EINVAL


def good():
    return dict(q=tensor(2, 1, 5, 128), k=tensor(2, 3, 7, 64, data=0x20000), v=tensor(2, 3, 7, 64, data=0x30000), y=tensor(2, 1, 5, 128, data=0x40000), mask=None)


@pytest.mark.parametrize("change", [
    dict(q=tensor(2, 1, 5, 120)), dict(k=tensor(2, 3, 7, 128, data=0x20000)), dict(v=tensor(2, 3, 6, 64, data=0x30000)), dict(y=tensor(2, 5, 1, 128, data=0x40000)),
    dict(y=tensor(2, 1, 5, 128, data=0x10000)), dict(y=tensor(2, 1, 5, 128, data=0x20000)), dict(y=tensor(2, 1, 5, 128, data=0x30000)),
    dict(k=tensor(3, 3, 7, 64, data=0x20000), v=tensor(3, 3, 7, 64, data=0x30000)), dict(k=tensor(1, 3, 7, 64, data=0x20000)),
    dict(q=tensor(2, 1, 5, 128, dn.F32)), dict(q=tensor(2, 1, 5, 128, data=0)), dict(q=tensor(2, 1, 0, 128)),
    dict(mask=dn.AttentionMask(0x50001, None, 0, 0)), dict(mask=dn.AttentionMask(None, 0x50001, -1, 0)), dict(mask=dn.AttentionMask(None, 0x50001, 0, -21))])
def test_attention_calls_that_are_refused(change):
    L, h = dn.lib(), C.c_void_p()
    dn.check(L.dnb_attention_plan_create(C.byref(dn.AttentionDesc(4, 2, 32, 0.0)), C.byref(h)))
    a = {**good(), **change}
    call = lambda plan, a: L.dnb_attention_forward(plan, C.byref(a["q"]), C.byref(a["k"]), C.byref(a["v"]), None if a["mask"] is None else C.byref(a["mask"]), C.byref(a["y"]), None)  # noqa: E731
    assert call(h, a) == dn.EINVAL
    assert b"attention" in L.dnb_last_error()
    assert call(None, good()) == dn.EINVAL
    assert L.dnb_attention_plan_set_diagnostics(h, -1, 0) == dn.EINVAL and L.dnb_attention_plan_set_diagnostics(h, 0, 1) == dn.EINVAL
    L.dnb_attention_plan_destroy(h)


def norm_call(L, x, residual=None, gain=None, eps=1e-6, total=None, y=None, q=None):
    ref = lambda t: None if t is None else C.byref(t)  # noqa: E731
    return L.dnb_rmsnorm_forward(ref(x), ref(residual), gain, eps, ref(total), ref(y), ref(q), None)


A, B = tensor(2, 3, 3, 60), tensor(2, 3, 3, 60, data=0x20000)
E = lambda data=0x30000, scales=0x40000, pitch=64, group=0: dn.E4M3(data, scales, pitch, group)  # noqa: E731


@pytest.mark.parametrize("a", [
    dict(x=None, y=B), dict(x=A), dict(x=A, y=B, total=tensor(2, 3, 3, 60, data=0x50000)), dict(x=A, y=tensor(2, 3, 3, 61, data=0x20000)),
    dict(x=A, y=tensor(2, 3, 3, 60, dn.F32, data=0x20000)), dict(x=A, residual=tensor(1, 3, 3, 60, data=0x20000), y=A), dict(x=A, residual=B, total=A, y=A),
    dict(x=A, y=tensor(2, 3, 3, 60, pitch=72)), dict(x=A, residual=B, y=tensor(2, 3, 3, 60, data=0x20000, pitch=72)), dict(x=A, y=B, eps=-1.0), dict(x=A, y=B, eps=math.nan),
    dict(x=A, y=B, gain=0x50002), dict(x=A, q=E(data=0)), dict(x=A, q=E(scales=0)), dict(x=A, q=E(pitch=56)), dict(x=A, q=E(pitch=66)), dict(x=A, q=E(group=48)),
    dict(x=A, q=E(group=-32)), dict(x=A, q=E(data=0x30004)), dict(x=A, q=E(data=0x10000)), dict(x=A, y=B, q=E(scales=0x20000)),
    dict(x=tensor(1, 2, 2, 8, dn.F32, layout=dn.NCHW), y=tensor(1, 2, 2, 8, dn.F32, data=0x20000, layout=dn.NCHW))])
def test_norm_calls_that_are_refused(a):
    L = dn.lib()
    assert norm_call(L, **a) == dn.EINVAL
    assert b"rmsnorm" in L.dnb_last_error()


def test_norm_of_too_many_channels_is_unsupported():
    L = dn.lib()
    assert norm_call(L, tensor(1, 1, 1, 32776), y=tensor(1, 1, 1, 32776, data=0x200000)) == dn.EUNSUPPORTED
    assert norm_call(L, tensor(1, 1, 1, 16392, dn.F32), y=tensor(1, 1, 1, 16392, dn.F32, data=0x200000)) == dn.EUNSUPPORTED


def test_binding_refuses_arrays_of_another_kind():
    import torch
    rope = dn.RopePlan(64, 2, (8, 12, 12))
    x, y = tensor(1, 4, 4, 128), tensor(1, 4, 4, 128, data=0x20000)
    with pytest.raises(ValueError, match="positions"):
        rope.forward(x, y, positions=torch.zeros(16, 3, dtype=torch.int32))     # not on a device
    attention = dn.CrossAttentionPlan(4, 2, 32)
    a = good()
    with pytest.raises(ValueError, match="lengths"):
        attention.forward(a["q"], a["k"], a["v"], a["y"], lengths=torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError, match="mask"):
        attention.forward(a["q"], a["k"], a["v"], a["y"], mask=torch.ones(2, 5, 21, dtype=torch.bool))
    with pytest.raises(ValueError, match="gain"):
        dn.rmsnorm(A, B, torch.ones(60), stream=0)
