"""Root-mean-square norm of more tokens than its blocks hold at once: every kernel's second and later tokens, against 64 bits."""
import pytest
import torch

import darknet_b200 as dn
from attention_util import HALF, norm_error
from test_gpu_attention import TORCH

pytestmark = pytest.mark.gpu

# 16-byte vectors of a token (32, 64, 128: a warp a token, 1, 2 or 4 vectors a thread; 256, 512: four warps; 1024: eight; above: 32), tokens: more than
# what 148 SMs take in one pass (148 * 32 of the first three, 148 * 8, 148 * 4, 148)
TOKENS = [(32, 9600), (64, 9600), (128, 9600), (256, 2500), (512, 2500), (1024, 1300), (2048, 400), (4096, 320)]


def within(got, want, bound, label):
    off = (got.double() - want).abs()
    assert bool(torch.isfinite(got.double()).all()), f"{label}: not finite"
    assert bool((off <= bound).all()), f"{label}: {int((off > bound).sum())} of {off.numel()} outside, worst {float((off - bound).max())}"


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("vecs,tokens", TOKENS)
@pytest.mark.parametrize("less", [0, 13])
@pytest.mark.parametrize("group", [None, 0, 32, 128])
def test_tokens_behind_the_first(dtype, vecs, tokens, less, group):
    """Neighbouring tokens differ in magnitude by up to 2^24, so that a sum, a largest value or a scale that is left from another token shows."""
    c = vecs * (8 if dtype == "bf16" else 4) - less
    c8 = (c + 7) // 8 * 8
    g = torch.Generator(device="cuda").manual_seed(vecs + less)
    size = 2.0 ** ((torch.arange(tokens, device="cuda") * 5 % 9) * 3 - 12).double()[:, None]
    x, r = (torch.zeros((1, 1, tokens, c8), dtype=TORCH[dtype], device="cuda") for _ in range(2))
    for t in (x, r):
        t[..., :c] = (torch.randn((tokens, c), generator=g, device="cuda") * size).to(TORCH[dtype])
    gain = torch.randn(c, generator=g, device="cuda")
    total, y = torch.full_like(x, 7.0), torch.full_like(x, 7.0)
    q = scales = None
    if group is not None:
        q = torch.full((1, 1, tokens, c8), 0x11, dtype=torch.uint8, device="cuda")
        scales = torch.full((1, 1, tokens, -(-c // group) if group else 1), -1.0, device="cuda")
    D = lambda t: dn.as_tensor(t, dn.NHWC, c)  # noqa: E731
    dn.rmsnorm(D(x), D(y), gain, 1e-6, D(r), D(total), q, scales, group or 0)
    s = x[0, 0, :, :c].double() + r[0, 0, :, :c].double()
    eps = float(torch.tensor(1e-6, dtype=torch.float32))
    want = s / ((s * s).mean(-1, keepdim=True) + eps).sqrt() * gain.double()
    e = norm_error(c)
    within(total[0, 0, :, :c], s, s.abs() * (HALF[dtype] + 2.0 ** -24), "sum")
    within(y[0, 0, :, :c], want, want.abs() * (HALF[dtype] + e), "norm")
    assert bool((y[..., c:] == 0).all()) and bool((total[..., c:] == 0).all())
    if group is None:
        return
    step = group or c
    padded = torch.nn.functional.pad(want, (0, scales.shape[-1] * step - c)).view(tokens, -1, step)
    scale = (padded.abs().amax(-1) / 448).clamp_min(2.0 ** -126)
    within(scales[0, 0], scale, scale * (e + 2.0 ** -23), "scales")
    got = scales[0, 0].double().repeat_interleave(step, -1)[:, :c]
    values = q[0, 0, :, :c].contiguous().view(torch.float8_e4m3fn).double() * got
    within(values, want, want.abs() * (2.0 ** -4 + 2 * e) + got * 2.0 ** -10, "8 bits")
    assert bool((q[..., c:] == 0).all())


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_squares_that_overflow(dtype):
    """Squares are fp32: 2^63 over 3 channels has a norm, 2^64 has zeros, with an infinity beside them NaN there."""
    x = torch.zeros((1, 1, 3, 8), dtype=TORCH[dtype], device="cuda")
    x[0, 0, 0, :3], x[0, 0, 1, :3] = 2.0 ** 63, 2.0 ** 64
    x[0, 0, 2, :3] = torch.tensor([2.0 ** 64, float("inf"), -1.0])
    y, q, scales = torch.full_like(x, 7.0), torch.full((1, 1, 3, 8), 0x11, dtype=torch.uint8, device="cuda"), torch.zeros((1, 1, 3, 1), device="cuda")
    dn.rmsnorm(dn.as_tensor(x, dn.NHWC, 3), dn.as_tensor(y, dn.NHWC, 3), None, 1e-6, e4m3=q, scales=scales)
    assert bool(((y[0, 0, 0, :3].double() - 1).abs() <= HALF[dtype] + norm_error(3)).all())
    assert bool((y[0, 0, 1] == 0).all()) and bool((q[0, 0, 1] == 0).all()) and scales[0, 0, 1].item() == 2.0 ** -126
    assert torch.isnan(y[0, 0, 2, :3]).tolist() == [False, True, False] and bool((y[0, 0, 2, [0, 2]] == 0).all()) and bool((y[..., 3:] == 0).all())
