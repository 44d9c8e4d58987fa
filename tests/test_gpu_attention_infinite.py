"""Cross attention of bf16 tensors with infinite queries: scores of -infinity weigh nothing, one of infinity makes NaN."""
import numpy as np
import pytest
import torch

import darknet_b200 as dn
from test_gpu_attention import device, empty, held, rng

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lq,heads,kv_heads,kernel", [(1, 4, 2, "rows_bf16"), (60, 4, 2, "tc_bf16"), (2, 130, 1, "simple")])
@pytest.mark.parametrize("scale", [0.3, -0.3])
def test_scores_of_infinity(lq, heads, kv_heads, kernel, scale):
    """Three images.  Queries of the first two are infinite in one channel, along which the first one's keys all make scores of -infinity (zeros, like a query
    that sees nothing) and one of the second's makes infinity (NaN); the third is finite."""
    n, keys, d = 3, 333, 64
    g = rng(lq)
    q, k, v = (held(g.standard_normal((n, 1, m, h * d)), "bf16") for m, h in ((lq, heads), (keys, kv_heads), (keys, kv_heads)))
    q[:2, ..., ::d] = np.inf
    k[:2, ..., ::d] = -np.sign(scale)
    k[1, 0, 200, ::d] = np.sign(scale)
    (_, qd), (_, kd), (_, vd) = keep = device(q, "bf16"), device(k, "bf16"), device(v, "bf16")
    yt, yd = empty(n, 1, lq, heads * d, "bf16")
    plan = dn.CrossAttentionPlan(heads, kv_heads, d, scale)
    plan.forward(qd, kd, vd, yd)
    plan.check_status()
    assert plan.kernel == kernel
    assert bool((yt[0] == 0).all()) and bool(torch.isnan(yt[1]).all()) and bool(torch.isfinite(yt[2]).all())
    mask = torch.ones((n, 1, keys), dtype=torch.bool, device="cuda")
    mask[1, 0, 200] = False                                      # the key that made NaN is hidden
    plan.forward(qd, kd, vd, yd, mask=mask.expand(n, lq, keys))
    assert bool((yt[:2] == 0).all()) and bool(torch.isfinite(yt[2]).all())
    del keep
