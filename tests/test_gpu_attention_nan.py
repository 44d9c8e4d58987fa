"""Cross attention of tensors that hold what is no number: it reaches the queries that see it, and no others."""
import numpy as np
import pytest
import torch

import darknet_b200 as dn
from attention_util import attention, attention_bound
from test_gpu_attention import device, empty, held, inside, rng

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("d,lq,heads,kv_heads", [(64, 1, 8, 2), (64, 3, 4, 4), (64, 40, 4, 2), (128, 150, 2, 2), (40, 300, 3, 1), (64, 2, 130, 1)])
@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_no_number_stays_with_the_queries_that_see_it(dtype, d, lq, heads, kv_heads, bad):
    """A query's channel, and keys that masks hide from some queries, in the first and in the last tile of keys."""
    n, kh, kw = 2, 20, 25
    lk = kh * kw
    g = rng(lq * 10 + d)
    q = held(g.standard_normal((n, 1, lq, heads * d)), dtype)
    k, v = (held(g.standard_normal((n, kh, kw, kv_heads * d)), dtype) for _ in range(2))
    mask = g.random((n, lq, lk)) < 0.6
    bad_keys = [3, lk - 2]
    mask[:, :, bad_keys] = g.random((n, lq, 2)) < 0.3
    if lq == 1:
        mask[0, 0, bad_keys], mask[1, 0, bad_keys] = False, [False, True]
    marked = k.reshape(n, lk, -1).copy()
    marked[:, bad_keys, 0] = bad                                  # of the first key head
    spoiled = q.copy()
    spoiled[0, 0, lq - 1, (heads - 1) * d] = np.nan               # the last query's last head
    (_, qd), (_, kd), (_, vd) = keep = device(spoiled, dtype), device(marked.reshape(k.shape), dtype), device(v, dtype)
    yt, yd = empty(n, 1, lq, heads * d, dtype)
    mt = torch.from_numpy(mask).cuda()
    plan = dn.CrossAttentionPlan(heads, kv_heads, d)
    plan.forward(qd, kd, vd, yd, mask=mt)
    plan.check_status()
    got = yt[:, 0].double().cpu().numpy().reshape(n, lq, heads, d)
    want, amount, size = attention(q[:, 0], k.reshape(n, lk, -1), v.reshape(n, lk, -1), heads, kv_heads, mask)
    bound = (attention_bound(want, amount, size, d, lk, dtype) + 1e-30).reshape(got.shape)
    reached = np.zeros((n, lq, heads), bool)
    # an infinite score is a weight of zero or no number, as its sign has it: only rows without one have a value to compare with
    reached[:, :, :heads // kv_heads] = mask[:, :, bad_keys].any(-1)[:, :, None]
    if np.isnan(bad):
        assert np.isnan(got[reached]).all()
    reached[0, lq - 1, heads - 1] |= mask[0, lq - 1].any()
    assert np.isnan(got[0, lq - 1, heads - 1]).all() or not mask[0, lq - 1].any()
    inside(got[~reached], want.reshape(got.shape)[~reached], bound[~reached], plan.kernel)
    del keep
