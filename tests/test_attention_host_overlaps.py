"""Outputs of rotary positions, cross attention and norm over positions, lengths, masks and gains are refused; checked without a GPU: the pointers are made-up
numbers, and a call that goes through fails for want of a device."""
import ctypes as C

import pytest

import darknet_b200 as dn

OUT, ROW, ROWS = 0x100000, 128, 24                       # the output: 2 x 3 x 4 tokens of 64 bf16 channels
END = OUT + ROWS * ROW


@pytest.fixture(autouse=True)
def no_device():
    import torch
    if torch.cuda.is_available():
        pytest.skip("made-up pointers")


def tensor(data, n=2, h=3, w=4, c=64):
    return dn.Tensor(data, dn.NHWC, dn.BF16, n, c, h, w, c)


def edges(size):
    """(address of `size` bytes, whether it reaches into the output): beside it on both sides, four bytes over each edge, inside, around it."""
    return [(OUT - size, False), (END, False), (OUT - size + 4, True), (END - 4, True), (OUT + 8, True), (OUT, True)]


def outcome(status, shared):
    assert status == (dn.EINVAL if shared else status) and status != dn.OK, dn.lib().dnb_last_error()
    assert shared or status != dn.EINVAL, dn.lib().dnb_last_error()
    assert not shared or b"memory" in dn.lib().dnb_last_error()


@pytest.mark.parametrize("at,shared", edges(ROWS * 12))
def test_positions_under_an_output(at, shared):
    L, rope, x, y = dn.lib(), C.c_void_p(), tensor(0x10000), tensor(OUT)
    d = dn.RopeDesc(64, 1, (C.c_int * 3)(0, 16, 16), 1, (C.c_int * 3)(0, 0, 0), 0, 1, 10000.0, (C.c_float * 3)(1.0, 1.0, 1.0))
    dn.check(L.dnb_rope_plan_create(C.byref(d), C.byref(rope)))
    outcome(L.dnb_rope_forward(rope, C.byref(x), at, C.byref(y), None), shared)
    outcome(L.dnb_rope_forward(rope, C.byref(y), at, C.byref(y), None), shared)         # in place
    L.dnb_rope_plan_destroy(rope)


@pytest.mark.parametrize("at,shared", edges(64 * 4))
@pytest.mark.parametrize("where", ["sum", "y", "values", "scales"])
def test_gains_under_an_output(at, shared, where):
    L, x, r, y = dn.lib(), tensor(0x10000), tensor(0x20000), tensor(OUT)
    B = C.byref
    if where == "sum":
        outcome(L.dnb_rmsnorm_forward(B(x), B(r), at, 1e-6, B(y), None, None, None), shared)
    elif where == "y":
        outcome(L.dnb_rmsnorm_forward(B(x), None, at, 1e-6, None, B(y), None, None), shared)
    elif where == "values":                                 # 24 rows of 64 bytes in a pitch of 128, the last of which ends early
        e = dn.E4M3(OUT, 0x300000, 128, 0)
        outcome(L.dnb_rmsnorm_forward(B(x), None, at - 64 if at == END or at == END - 4 else at, 1e-6, None, None, B(e), None), shared)
    else:
        e = dn.E4M3(0x300000, END - ROWS * 8, 64, 32)      # two scales a token, that end where the output of the other cases does
        at = {OUT - 256: END - ROWS * 8 - 256, OUT - 252: END - ROWS * 8 - 252, OUT + 8: END - ROWS * 8 + 8, OUT: END - ROWS * 8}.get(at, at)
        outcome(L.dnb_rmsnorm_forward(B(x), None, at, 1e-6, None, None, B(e), None), shared)


def attend(mask):
    L, plan = dn.lib(), C.c_void_p()
    dn.check(L.dnb_attention_plan_create(C.byref(dn.AttentionDesc(1, 1, 64, 0.0)), C.byref(plan)))
    q, k, v, y = tensor(0x10000), tensor(0x20000, h=5, w=6), tensor(0x30000, h=5, w=6), tensor(OUT)
    status = L.dnb_attention_forward(plan, C.byref(q), C.byref(k), C.byref(v), C.byref(mask), C.byref(y), None)
    L.dnb_attention_plan_destroy(plan)
    return status


@pytest.mark.parametrize("at,shared", edges(8))
def test_lengths_under_an_output(at, shared):
    outcome(attend(dn.AttentionMask(at, None, 0, 0)), shared)


# a mask of 2 images x 12 queries x 30 keys: its address, strides, and whether the output lies on one of its rows
MASKS = [(OUT - 2 * 12 * 30, 360, 30, False), (OUT - 2 * 12 * 30 + 1, 360, 30, True), (END, 360, 30, False), (END - 1, 360, 30, True), (OUT + 100, 360, 30, True),
         (OUT - 360, 0, 30, False), (OUT - 359, 0, 30, True), (OUT - 30, 0, 0, False), (OUT - 29, 0, 0, True), (END - 1, 0, 0, True),
         # rows far apart, around the output or on it
         (OUT - 30, ROWS * ROW + 30, 0, False), (OUT - 30, ROWS * ROW + 29, 0, True), (OUT - 30, 0, ROWS * ROW + 30, False), (OUT - 30, 0, ROWS * ROW + 29, True),
         (OUT - 11 * 0x10000 - 30, 0, 0x10000, False), (OUT - 11 * 0x10000 - 29, 0, 0x10000, True), (OUT - 5 * 0x1000 - 30, 0, 0x1000, False), (OUT - 5 * 0x1000, 0, 0x1000, True),
         (OUT - 0x8000, 0x9000, 1, False), (OUT - 0x8000, 0x8000, 1, True), (OUT - 0x8000, 0x8000 - 40, 1, True), (OUT - 0x8000, 0x8000 - 41, 1, False),
         (OUT - 100, 2 ** 63 - 1, 2 ** 63 - 1, False), (OUT - 10, 2 ** 63 - 1, 2 ** 63 - 1, True), (0x40000, 2 ** 63 - 1, 0, False)]


@pytest.mark.parametrize("at,image,query,shared", MASKS)
def test_masks_under_an_output(at, image, query, shared):
    outcome(attend(dn.AttentionMask(None, at, image, query)), shared)
    rows = [at + i * image + j * query for i in range(2) for j in range(12)]
    assert shared == any(r < END and r + 30 > OUT for r in rows)        # what the case says of itself


def test_strides_of_a_single_image_and_query_do_not_count():
    L, plan = dn.lib(), C.c_void_p()
    dn.check(L.dnb_attention_plan_create(C.byref(dn.AttentionDesc(1, 1, 64, 0.0)), C.byref(plan)))
    q, k, v, y = tensor(0x10000, 1, 1, 1), tensor(0x20000, 1), tensor(0x30000, 1), tensor(OUT, 1, 1, 1)
    m = dn.AttentionMask(None, OUT - 12, 1 << 40, 1 << 40)
    outcome(L.dnb_attention_forward(plan, C.byref(q), C.byref(k), C.byref(v), C.byref(m), C.byref(y), None), False)
    L.dnb_attention_plan_destroy(plan)
