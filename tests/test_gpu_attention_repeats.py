"""Cross attention gives the same bits whatever ran before it: rows of a tile that no query fills hold what earlier kernels left in shared memory."""
import numpy as np
import pytest
import torch

import darknet_b200 as dn
from test_gpu_attention import attend, rng

pytestmark = pytest.mark.gpu

D = lambda t: dn.as_tensor(t, dn.NHWC)  # noqa: E731


def leave_behind(value, d):
    """Every SM's shared memory filled with `value`: queries, keys and values of two calls over more tiles than the GPU has SMs."""
    for lq in (256, 256):
        q, k = torch.full((74, 1, lq, 4 * d), value, device="cuda").bfloat16(), torch.full((74, 38, 38, 4 * d), value, device="cuda").bfloat16()
        dn.CrossAttentionPlan(4, 4, d).forward(D(q), D(k), D(k), D(torch.empty_like(q)))
    torch.cuda.synchronize()


@pytest.mark.parametrize("d", [40, 64, 128])
@pytest.mark.parametrize("heads,kv_heads", [(3, 1), (12, 4), (5, 1), (14, 2), (100, 1)])
@pytest.mark.parametrize("masked", [False, True])
def test_rows_that_no_query_fills(d, heads, kv_heads, masked):
    """Heads of a key head that 128 is no multiple of, over several tiles of keys, so that the running maximum may move or stay."""
    mask = rng(heads + d).random((2, 90, 30 * 31)) < 0.7 if masked else None
    plan, (qt, kt, vt, yt) = attend("bf16", 2, 90, 30, 31, heads, kv_heads, d, mask=mask)
    assert plan.kernel == "tc_bf16"
    mt = None if mask is None else torch.from_numpy(mask).cuda()
    first = None
    for value in (0.0, np.nan, 1.0, -1e30, np.inf):
        leave_behind(value, 128 if d > 64 else 64)
        yt.fill_(3.0)
        plan.forward(*(D(t) for t in (qt, kt, vt, yt)), mask=mt)
        torch.cuda.synchronize()
        plan.check_status()
        first = yt.clone() if first is None else first
        assert torch.equal(first, yt), f"after {value}: {int((first != yt).sum())} values differ"
