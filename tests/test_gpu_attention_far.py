"""Cross attention whose masks, queries and outputs lie more than 2^31 bytes or elements apart."""
import numpy as np
import pytest
import torch

import darknet_b200 as dn
from attention_util import attention, attention_bound
from test_gpu_attention import TORCH, attend, device, empty, held, inside, rng

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("lq,heads,kv_heads", [(1, 4, 2), (3, 4, 2), (70, 4, 2), (2, 130, 1)])
@pytest.mark.parametrize("rows", [False, True])
def test_masks_whose_rows_are_far_apart(dtype, lq, heads, kv_heads, rows):
    """Images 1.6e9 bytes apart, or an image's queries as far as that lets them be, in a buffer of ones."""
    n, keys, d = 3, 150, 40
    apart = 1_600_000_007
    step = (apart - keys) // lq if rows else keys
    buffer = torch.ones(2 * apart + lq * step + keys, dtype=torch.uint8, device="cuda")
    mask = buffer.as_strided((n, lq, keys), (apart, step, 1))
    g = rng(lq + 17)
    allowed = g.random((n, lq, keys)) < 0.5
    mask.copy_(torch.from_numpy(allowed).cuda())
    q = held(g.standard_normal((n, 1, lq, heads * d)), dtype)
    k, v = (held(g.standard_normal((n, 1, keys, kv_heads * d)), dtype) for _ in range(2))
    (_, qd), (_, kd), (_, vd) = keep = device(q, dtype), device(k, dtype), device(v, dtype)
    yt, yd = empty(n, 1, lq, heads * d, dtype)
    plan = dn.CrossAttentionPlan(heads, kv_heads, d)
    plan.forward(qd, kd, vd, yd, mask=mask)
    plan.check_status()
    want, amount, size = attention(q[:, 0], k[:, 0], v[:, 0], heads, kv_heads, allowed)
    inside(yt[:, 0], want, attention_bound(want, amount, size, d, keys, dtype) + 1e-30, plan.kernel)
    del keep


@pytest.mark.parametrize("dtype,heads,kv_heads", [("bf16", 8, 8), ("bf16", 8, 1), ("f32", 8, 8), ("bf16", 256, 1), ("f32", 256, 1)])
def test_queries_and_outputs_behind_32_bits(dtype, heads, kv_heads):
    """One image of more than 2^31 elements: its first and last queries."""
    d, keys = max(8, 1024 // heads), 12
    c = heads * d
    lq = 2 ** 31 // c + 70
    q = torch.zeros((1, 1, lq, c), dtype=TORCH[dtype], device="cuda")
    assert q.numel() > 2 ** 31
    some = [0, 1, lq - 71, lq - 2, lq - 1]
    g = rng(d)
    x = held(g.standard_normal((len(some), c)), dtype)
    q[0, 0, some] = torch.from_numpy(x).to("cuda", TORCH[dtype])
    k, v = (held(g.standard_normal((1, 1, keys, kv_heads * d)), dtype) for _ in range(2))
    (_, kd), (_, vd) = keep = device(k, dtype), device(v, dtype)
    y = torch.full_like(q, 7.0)
    plan = dn.CrossAttentionPlan(heads, kv_heads, d)
    plan.forward(dn.as_tensor(q, dn.NHWC), kd, vd, dn.as_tensor(y, dn.NHWC))
    plan.check_status()
    want, amount, size = attention(x[None], k[:, 0], v[:, 0], heads, kv_heads, np.ones((1, len(some), keys), bool))
    inside(y[0, 0, some][None], want, attention_bound(want, amount, size, d, keys, dtype), plan.kernel)
    mean = y[0, 0, 2]                                             # queries of zeros weigh all keys alike
    others = torch.ones(lq, dtype=torch.bool, device="cuda")
    others[some] = False
    for first in range(0, lq, 1 << 18):
        part = y[0, 0, first:first + (1 << 18)]
        assert bool((part == mean).all(-1)[others[first:first + (1 << 18)]].all())
    del keep
