"""Cross attention whose waits run out early in a long walk over the keys, in blocks of a cluster too: every role ends, the call is reported, the next one is right."""
import pytest
import torch

import darknet_b200 as dn
from test_gpu_attention import TORCH

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("n,lq,d", [(2, 1, 64), (2, 1, 128), (40, 2, 64), (2, 200, 64), (2, 200, 128), (40, 200, 64), (40, 200, 128)])
@pytest.mark.parametrize("masked", [False, True])
def test_a_wait_that_runs_out_before_many_tiles(dtype, n, lq, d, masked):
    heads, side = 4, 38
    g = torch.Generator(device="cuda").manual_seed(lq + d)
    q, k, v = (torch.randn((n, h, w, heads * d), generator=g, device="cuda").to(TORCH[dtype]) for h, w in ((1, lq), (side, side), (side, side)))
    mask = torch.rand((n, lq, side * side), generator=g, device="cuda") < 0.9 if masked else None
    y = torch.zeros_like(q)
    D = [dn.as_tensor(t, dn.NHWC) for t in (q, k, v, y)]
    plan = dn.CrossAttentionPlan(heads, heads, d)
    plan.forward(*D, mask=mask)
    plan.check_status()
    want = y.clone()
    plan.set_diagnostics(wait_limit_cycles=400_000, debug_bits=32)
    for _ in range(2):
        plan.forward(*D, mask=mask)
        with pytest.raises(dn.DarknetB200Error, match="wait") as e:
            plan.check_status()
        assert e.value.status == dn.ETIMEOUT
    plan.set_diagnostics()
    y.zero_()
    plan.forward(*D, mask=mask)
    plan.check_status()
    assert torch.equal(y, want)
