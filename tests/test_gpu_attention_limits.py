"""Cross attention where its kernels' tiles, copies and waits end: masks that start at any byte, keys up to a tile's border, query heads that fill a tile,
sums of far apart values in f32, a first call inside a capture, and waits that run out."""
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

import darknet_b200 as dn
from attention_util import attention, attention_bound
from test_gpu_attention import TORCH, attend, device, empty, held, inside, rng

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("lq", [1, 60])
@pytest.mark.parametrize("keys", [1, 15, 16, 17, 63, 65, 127, 130, 301])
@pytest.mark.parametrize("offset", [0, 1, 7, 15])
def test_masks_that_start_at_any_byte(dtype, lq, keys, offset):
    """A mask in the middle of other bytes, all of them set: none of those shows through, and bytes other than 0 and 1 count."""
    n, heads, kv_heads, d = 2, 4, 2, 40
    g = rng(keys * 100 + offset)
    q, k, v = held(g.standard_normal((n, 1, lq, heads * d)), dtype), held(g.standard_normal((n, 1, keys, kv_heads * d)), dtype), held(g.standard_normal((n, 1, keys, kv_heads * d)), dtype)
    allowed = g.random((n, lq, keys)) < 0.5
    buffer = torch.full((offset + n * lq * keys + 64,), 255, dtype=torch.uint8, device="cuda")
    mask = buffer[offset:offset + n * lq * keys].view(n, lq, keys)
    values = np.where(allowed, g.choice(np.array([1, 2, 128, 255], np.uint8), allowed.shape), 0).astype(np.uint8)
    mask.copy_(torch.from_numpy(values).cuda())
    (_, qd), (_, kd), (_, vd) = keep = device(q, dtype), device(k, dtype), device(v, dtype)
    yt, yd = empty(n, 1, lq, heads * d, dtype)
    plan = dn.CrossAttentionPlan(heads, kv_heads, d)
    plan.forward(qd, kd, vd, yd, mask=mask)
    plan.check_status()
    want, amount, size = attention(q[:, 0], k[:, 0], v[:, 0], heads, kv_heads, allowed)
    inside(yt[:, 0], want, attention_bound(want, amount, size, d, keys, dtype) + 1e-30, plan.kernel)
    del keep


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("heads,kv_heads", [(17, 1), (63, 1), (64, 1), (65, 1), (100, 1), (127, 1), (128, 1), (129, 1), (256, 2)])
@pytest.mark.parametrize("lq", [1, 3])
def test_heads_that_fill_a_tile(dtype, heads, kv_heads, lq):
    attend(dtype, 2, lq, 11, 13, heads, kv_heads, 16)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("n,heads,lq,keys", [(1, 1, 40, (76, 76)), (19, 8, 129, (38, 38)), (40, 4, 17, (30, 31)), (1, 8, 40, (25, 41)), (3, 5, 300, (50, 41))])
def test_splits_of_the_keys(dtype, n, heads, lq, keys):
    """One job and many, whose keys one, two, four or eight blocks share."""
    attend(dtype, n, lq, *keys, heads, heads, 64, lengths=[keys[0] * keys[1] - 37 * i for i in range(n)])


@pytest.mark.parametrize("lq", [1, 40])
@pytest.mark.parametrize("exponent", [-60, 0, 60])
def test_f32_keeps_24_bits(lq, exponent):
    """Values of any size between 2^-109 and 2^127 lose nothing by their split into three parts: equal weights, values that the tensor cores' parts have to
    carry to the last bit.  One key each: the output is the value itself."""
    heads, d = 4, 64
    g = rng(exponent + 200)
    v = held(g.standard_normal((2, 1, 1, heads * d)) * 2.0 ** exponent, "f32")
    q, k = (held(g.standard_normal((2, 1, m, heads * d)), "f32") for m in (lq, 1))
    (_, qd), (_, kd), (_, vd) = keep = device(q, "f32"), device(k, "f32"), device(v, "f32")
    yt, yd = empty(2, 1, lq, heads * d, "f32")
    dn.CrossAttentionPlan(heads, heads, d).forward(qd, kd, vd, yd)
    # six parts' products onto one another, smallest first, an add each that may cut instead of rounding (2^-23), and the last quotient
    assert (np.abs(yt[:, 0].double().cpu().numpy() - v[:, 0]) <= np.abs(v[:, 0]) * 8 * 2.0 ** -23).all()
    del keep


@pytest.mark.parametrize("dtype,lq,d", [("bf16", 1, 64), ("bf16", 1, 128), ("f32", 1, 64), ("f32", 1, 128), ("bf16", 200, 64), ("bf16", 200, 128), ("f32", 200, 64), ("f32", 200, 128)])
def test_a_wait_that_runs_out_is_reported(dtype, lq, d):
    """One load is left out: the call ends, check_status says so, once, and the next call is right."""
    n, heads, side = 2, 2, 13
    q, k, v = (torch.randn((n, h, w, heads * d), device="cuda").to(TORCH[dtype]) for h, w in ((1, lq), (side, side), (side, side)))
    y = torch.zeros_like(q)
    D = [dn.as_tensor(t, dn.NHWC) for t in (q, k, v, y)]
    plan = dn.CrossAttentionPlan(heads, heads, d)
    plan.forward(*D)
    plan.check_status()
    want = y.clone()
    plan.set_diagnostics(wait_limit_cycles=2_000_000, debug_bits=32)
    plan.forward(*D)
    with pytest.raises(dn.DarknetB200Error, match="wait") as e:
        plan.check_status()
    assert e.value.status == dn.ETIMEOUT
    plan.check_status()
    plan.set_diagnostics()
    y.zero_()
    plan.forward(*D)
    plan.check_status()
    assert torch.equal(y, want)


FIRST = """
import torch, darknet_b200 as dn
dtype, lq = torch.{dtype}, {lq}
q, k, v = (torch.randn((2, h, w, 256), device="cuda").to(dtype) for h, w in ((1, lq), (13, 13), (13, 13)))
y = torch.zeros_like(q)
plan = dn.CrossAttentionPlan(4, 4, 64)
D = [dn.as_tensor(t, dn.NHWC) for t in (q, k, v, y)]
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    plan.forward(*D)
graph.replay()
torch.cuda.synchronize()
got = y.clone()
plan.forward(*D)
plan.check_status()
assert got.abs().sum() > 0 and torch.equal(got, y)
"""


@pytest.mark.parametrize("dtype,lq", [("bfloat16", 40), ("float32", 40), ("float32", 1)])
def test_a_first_call_inside_a_capture(dtype, lq):
    """Nothing has to have run before: a process whose first call of a kernel is captured."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    subprocess.run([sys.executable, "-c", FIRST.format(dtype=dtype, lq=lq)], check=True, cwd=root, timeout=300)
