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
