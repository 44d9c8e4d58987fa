"""Limits of cross attention's entry point, checked without a GPU: the pointers are made-up numbers, and each call ends before anything is launched."""
import ctypes as C

import pytest

import darknet_b200 as dn


def tensor(n, h, w, c, data):
    return dn.Tensor(data, dn.NHWC, dn.BF16, n, c, h, w, c)


@pytest.mark.parametrize("queries,keys", [((1, 5), (1 << 15, (1 << 15) + 1)), (((1 << 30) + 1, 1), (3, 7)), ((1, 5), (1, 2 ** 31 - 1))])
def test_more_tokens_than_a_tile_count_holds(queries, keys):
    L, h = dn.lib(), C.c_void_p()
    dn.check(L.dnb_attention_plan_create(C.byref(dn.AttentionDesc(1, 1, 8, 0.0)), C.byref(h)))
    q, y = (tensor(1, *queries, 8, at) for at in (1 << 40, 2 << 40))
    k, v = (tensor(1, *keys, 8, at) for at in (3 << 40, 4 << 40))
    assert L.dnb_attention_forward(h, C.byref(q), C.byref(k), C.byref(v), None, C.byref(y), None) == dn.EUNSUPPORTED
    assert b"tokens" in L.dnb_last_error()
    L.dnb_attention_plan_destroy(h)


def ranged(data, c, pitch, n=2, h=3, w=4, dtype=None):
    return dn.Tensor(data, dn.NHWC, dn.BF16 if dtype is None else dtype, n, c, h, w, pitch)


# the output's place beside an input of 2 x 3 x 4 x 64 bf16 at 0x10000, 128 or 256 bytes a row; whether they share memory
PLACES = [(128, 0x10000 + 128, False), (128, 0x10000 - 128, False), (64, 0x10000 + 128, True), (64, 0x10000 + 24 * 128, False), (64, 0x10000 - 24 * 128, False),
          (64, 0x10000 - 23 * 128, True), (128, 0x10000 + 23 * 256 + 128, False), (128, 0x10000 + 23 * 256, True), (192, 0x10000 + 256, False), (96, 0x10000 + 128, True)]


@pytest.mark.parametrize("pitch,at,shared", PLACES)
def test_outputs_beside_their_inputs(pitch, at, shared):
    """Channel ranges of one wider tensor beside one another go through (and fail for want of a device only); what overlaps is refused."""
    import torch
    if torch.cuda.is_available():
        pytest.skip("made-up pointers")
    L, rope, attention = dn.lib(), C.c_void_p(), C.c_void_p()
    x, y = ranged(0x10000, 64, pitch), ranged(at, 64, pitch)
    status = L.dnb_rmsnorm_forward(C.byref(x), None, None, 1e-6, None, C.byref(y), None, None)
    assert (status == dn.EINVAL) == shared, L.dnb_last_error()
    d = dn.RopeDesc(64, 1, (C.c_int * 3)(0, 16, 16), 1, (C.c_int * 3)(0, 0, 0), 0, 1, 10000.0, (C.c_float * 3)(1.0, 1.0, 1.0))
    dn.check(L.dnb_rope_plan_create(C.byref(d), C.byref(rope)))
    assert (L.dnb_rope_forward(rope, C.byref(x), None, C.byref(y), None) == dn.EINVAL) == shared
    L.dnb_rope_plan_destroy(rope)
    dn.check(L.dnb_attention_plan_create(C.byref(dn.AttentionDesc(1, 1, 64, 0.0)), C.byref(attention)))
    far = ranged(0x90000, 64, pitch)
    assert (L.dnb_attention_forward(attention, C.byref(far), C.byref(x), C.byref(far), None, C.byref(y), None) == dn.EINVAL) == shared
    L.dnb_attention_plan_destroy(attention)


@pytest.mark.parametrize("data,scales,refused", [(0x20000, 0x30000, False), (0x10000 + 23 * 128, 0x30000, True), (0x20000, 0x10000 - 24 * 4 + 4, True), (0x20000, 0x20000 + 24 * 64 - 4, True),
                                                 (0x20000, 0x20000 + 24 * 64, False), (0x10000 + 24 * 128, 0x10000 - 24 * 4, False)])
def test_e4m3_outputs_beside_the_others(data, scales, refused):
    import torch
    if torch.cuda.is_available():
        pytest.skip("made-up pointers")
    L, x, q = dn.lib(), ranged(0x10000, 64, 64), dn.E4M3(data, scales, 64, 0)
    assert (L.dnb_rmsnorm_forward(C.byref(x), None, None, 1e-6, None, None, C.byref(q), None) == dn.EINVAL) == refused, L.dnb_last_error()
