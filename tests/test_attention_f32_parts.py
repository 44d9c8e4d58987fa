"""Cross attention of f32 tensors keeps 24 bits of every operand: calls whose result hangs on the third bf16 part of queries, keys, weights and values, and on
each of the six products of parts.  On the CPU an emulation shows that each loss is outside the bounds that the kernels are held to."""
import numpy as np
import pytest

SIX = ((2, 0), (0, 2), (1, 1), (1, 0), (0, 1), (0, 0))       # parts of (query, key) or (weight, value): 0 the highest
BIG = 64.0                                                   # scores of 64 * 64


def bf16(x):
    """The nearest bf16 number, ties to even, of a float64 that fp32 holds."""
    u = np.asarray(x, np.float32).view(np.uint32).astype(np.uint64)
    return ((u + 0x7fff + (u >> 16 & 1)) >> 16 << 16).astype(np.uint32).view(np.float32).astype(np.float64)


def parts(x):
    hi = bf16(x)
    mid = bf16(x - hi)
    return hi, mid, bf16(x - hi - mid)


def product(a, b, kept=SIX):
    a, b = parts(a), parts(b)
    return sum(a[i] * b[j] for i, j in kept)


# Scores: two keys, each with a channel of its own, that differ by little: (q0, q1, k0, k1), in units of BIG.  MID: nothing in the highest part but 1, all in the
# middle one; LOW: 3/4 of half a step of the middle part.
MID, LOW = 2.0 ** -8 - 2.0 ** -15, 0.75 * 2.0 ** -17
SCORES = {
    "low part of the keys": (1.0, 1.0, 1 + 2.0 ** -9 + LOW, 1 + 2.0 ** -9),
    "low part of the queries": (1 + 2.0 ** -9 + LOW, 1 + 2.0 ** -9, 1.0, 1.0),
    "middle parts of both": (1 + MID, 1 + 2 * MID, 1 + MID, 1.0),
    "middle part of the queries": (1 + MID, 1.0, 1.0, 1.0),
    "middle part of the keys": (1.0, 1.0, 1.0, 1 + MID),
    "all parts": (1 + MID + LOW / 4, 1 + 2.0 ** -9 + LOW, 1 + 2.0 ** -9 + LOW, 1 + MID + LOW / 4)}
# A score of BIG * BIG: the three products left out (2^-8 2^-16 of it twice, and less), the last of the six additions, which may cut (2^-23, and 2^-7 of
# that for those before it), its product with the scale (2^-24): under 2^-21.5 of it, for each of two keys.  An output p0 - p1 = tanh(difference / 2) moves by half
# of what the difference does, and by the weights' own 2^-20.
SCORE_BOUND = 0.5 * 2 * BIG * BIG * 2.0 ** -21.5 * 1.01 + 2.0 ** -20


def score_inputs(case):
    q0, q1, k0, k1 = (np.float64(np.float32(BIG * v)) for v in SCORES[case])
    return q0, q1, k0, k1


# Weights and values: the larger weight is 1, the other e^-u, values 1 and -e^u as fp32 has it, so that the two products cancel.  Sixty-four u at once.
US = np.float64(np.float32(np.linspace(0.11, 0.93, 64)))
VALUES = np.float64(np.float32(-np.exp(US)))
# Each product over the sum of the weights is 1 / (1 + e^-u) < 1 or less.  The smaller weight's relative error: its exponential (2 ulp: 2^-22) and its score (u < 1:
# an addition that may cut, 2^-23, the product with the scale and the scale's own rounding, 2^-24 each).  Then the products left out (2^-23) and the additions
# that may cut (2^-23: the two keys' highest products, the parts before them, the sum of the tiles).
WEIGHT_BOUND = (2.0 ** -22 + 2.0 ** -22) + 2.0 ** -23 + 3 * 2.0 ** -23


def weighted(kept=SIX):
    p = np.float64(np.float32(np.exp(-US)))
    return (1.0 + product(p, VALUES, kept)) / (1.0 + p)


def test_two_parts_are_outside_the_bounds():
    """What any lost product of parts does to these calls, and what six of them do."""
    lost = {pair: 0.0 for pair in SIX}
    for case in SCORES:
        q0, q1, k0, k1 = score_inputs(case)
        want = np.tanh((q0 * k0 - q1 * k1) / 2)
        assert abs(np.tanh((product(q0, k0) - product(q1, k1)) / 2) - want) <= SCORE_BOUND
        for pair in SIX:
            kept = [s for s in SIX if s != pair]
            lost[pair] = max(lost[pair], abs(np.tanh((product(q0, k0, kept) - product(q1, k1, kept)) / 2) - want))
    assert all(off > 2 * SCORE_BOUND for off in lost.values()), lost
    p = np.exp(-US)
    want = (1.0 + p * VALUES) / (1.0 + p)
    assert (np.abs(weighted() - want) <= WEIGHT_BOUND).all()
    for pair in SIX:
        assert np.abs(weighted([s for s in SIX if s != pair]) - want).max() > 2 * WEIGHT_BOUND, pair


LQ = pytest.mark.parametrize("lq", [1, 16, 17, 200])          # up to 16 rows, and more: the two kernels
D = pytest.mark.parametrize("d", [8, 64, 128])


def call(q, k, v, scale):
    """q [lq, d], k, v [keys, d], of two heads that hold the same."""
    import torch

    import darknet_b200 as dn
    tensors = [torch.from_numpy(np.concatenate([t, t], -1).astype(np.float32)).cuda()[None, None].contiguous() for t in (q, k, v)]
    y = torch.empty_like(tensors[0])
    plan = dn.CrossAttentionPlan(2, 2, q.shape[1], scale)
    plan.forward(*(dn.as_tensor(t, dn.NHWC) for t in (*tensors, y)))
    plan.check_status()
    assert plan.kernel == ("rows_f32" if q.shape[0] <= 16 else "tc_f32")
    a, b = y[0, 0].double().cpu().numpy().reshape(q.shape[0], 2, -1).transpose(1, 0, 2)
    assert (a == b).all()
    return a


@pytest.mark.gpu
@pytest.mark.parametrize("case", SCORES)
@LQ
@D
def test_scores_that_hang_on_every_part(case, lq, d):
    q0, q1, k0, k1 = score_inputs(case)
    q, k, v = np.zeros((lq, d)), np.zeros((2, d)), np.zeros((2, d))
    q[:, 1], q[:, d - 2], k[0, 1], k[1, d - 2] = q0, q1, k0, k1
    v[0], v[1] = 1.0, -1.0
    assert np.abs(call(q, k, v, 1.0) - np.tanh((q0 * k0 - q1 * k1) / 2)).max() <= SCORE_BOUND


@pytest.mark.gpu
@LQ
@D
def test_weights_and_values_that_cancel(lq, d):
    for first in range(0, 64, lq):
        us = US[first:first + lq] if lq < 64 else np.resize(US, lq)
        values = np.float32(-np.exp(us)).astype(np.float64)
        rows = len(us)
        q, k, v = np.zeros((lq, d)), np.zeros((2, d)), np.ones((2, d))
        q[:rows, 3], k[0, 3], k[1, 3] = us, 0.0, -1.0
        channels = min(rows, d)                                # channel c: the value that cancels for row c
        v[1, :channels] = values[:channels]
        p = np.exp(-q[:, 3:4])
        want = (v[0] + p * v[1]) / (1.0 + p)
        got = call(q, k, v, 1.0)
        size = (np.abs(v[0]) + p * np.abs(v[1])) / (1.0 + p)  # of the two products together: 2 / (1 + p) where they cancel
        off = np.abs(got - want)
        # a result that is not near zero has the error of the sum of the weights and of the quotient, too (2^-21 of a weight, 2^-23 for two roundings and a sum)
        assert (off <= WEIGHT_BOUND * np.maximum(size, 1.0) + (2.0 ** -21 + 2.0 ** -22) * np.abs(want)).all(), float((off / size).max())
        if lq >= 64:
            break
