"""Scales of cross attention that the kernels can hold, checked without a GPU."""
import ctypes as C
import math

import pytest

import darknet_b200 as dn


@pytest.mark.parametrize("scale,taken", [(2.35e38, True), (-2.35e38, True), (1e-45, True), (2.37e38, False), (-3.4e38, False), (math.inf, False), (-math.inf, False), (math.nan, False)])
def test_scales_whose_product_with_log2_e_is_no_number(scale, taken):
    """Every score is multiplied by it: zero times infinity would make NaN of all."""
    L, h = dn.lib(), C.c_void_p()
    assert L.dnb_attention_plan_create(C.byref(dn.AttentionDesc(8, 8, 64, scale)), C.byref(h)) == (dn.OK if taken else dn.EINVAL)
    assert bool(h) == taken and (taken or b"scale" in L.dnb_last_error())
    L.dnb_attention_plan_destroy(h)
