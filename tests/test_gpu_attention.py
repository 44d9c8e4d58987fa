"""Rotary positions, cross attention and root-mean-square norm on the GPU against plain implementations in 64 bits (attention_util.py), each output
within the bound that the arithmetic of the kernels' types allows."""
import numpy as np
import pytest
import torch

import darknet_b200 as dn
from attention_util import HALF, attention, attention_bound, grid_positions, norm, norm_error, rope, rope_bound

pytestmark = pytest.mark.gpu

TORCH = {"bf16": torch.bfloat16, "f32": torch.float32}


def rng(seed):
    return np.random.Generator(np.random.Philox(key=[seed, 91]))


def held(a, dtype):
    """float64 values as the type holds them."""
    return torch.from_numpy(np.ascontiguousarray(a, np.float32)).to(TORCH[dtype]).double().numpy()


def device(a, dtype, pitch=None, fill=0.0):
    """[n, h, w, c] in float64 -> (device tensor of a pitch, dnb_tensor)."""
    n, h, w, c = a.shape
    t = torch.full((n, h, w, pitch or (c + 7) // 8 * 8), fill, dtype=TORCH[dtype], device="cuda")
    t[..., :(c + 7) // 8 * 8] = 0
    t[..., :c] = torch.from_numpy(a).to("cuda", TORCH[dtype])
    return t, dn.as_tensor(t, dn.NHWC, c)


def empty(n, h, w, c, dtype, pitch=None):
    t = torch.full((n, h, w, pitch or (c + 7) // 8 * 8), 7.0, dtype=TORCH[dtype], device="cuda")
    return t, dn.as_tensor(t, dn.NHWC, c)


def inside(got, want, bound, label=""):
    got = got.double().cpu().numpy() if hasattr(got, "cpu") else got
    off = np.abs(got - want)
    assert np.isfinite(got).all(), f"{label}: {np.count_nonzero(~np.isfinite(got))} values are not finite"
    worst = np.unravel_index(np.argmax(off - bound), off.shape)
    assert (off <= bound).all(), f"{label}: {np.count_nonzero(off > bound)} of {off.size} outside; at {worst}: {got[worst]} for {want[worst]}, bound {bound[worst]}"


# ------------------------------------------------------------------ rotary positions
ROPES = [  # n, h, w, c, heads, head_dim, pairs, interleaved, shared, given
    (1, 1, 1, 64, 1, 64, (8, 12, 12), False, True, True), (2, 5, 7, 200, 3, 64, (8, 12, 12), True, True, False), (4, 3, 9, 131, 2, 36, (2, 7, 9), False, False, False),
    (2, 4, 5, 40, 2, 18, (0, 4, 5), True, False, True), (3, 19, 25, 511, 7, 72, (0, 18, 18), True, False, False), (1, 2, 3, 256, 1, 256, (28, 50, 50), False, True, True),
    (2, 3, 3, 96, 4, 24, (0, 0, 8), False, True, False), (1, 6, 6, 10, 5, 2, (1, 0, 0), False, True, True), (1, 300, 1, 24, 3, 8, (1, 1, 1), True, True, False),
    (2, 9, 4, 21, 2, 6, (1, 1, 1), False, False, False)]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("case", ROPES)
def test_rope(case, dtype):
    n, h, w, c, heads, d, pairs, interleaved, shared, given = case
    g = rng(n * 1000 + c)
    x = held(g.standard_normal((n, h, w, c)), dtype)
    frames, origin, scale = (2 if n % 2 == 0 else 1), (3, -2, 100), (1.0, 0.5, 2.0)
    at = g.integers(-2 ** 31, 2 ** 31, (n * h * w, 3)) if given else grid_positions(n, h, w, frames, origin)
    plan = dn.RopePlan(d, heads, pairs, 10000.0, interleaved, shared, frames, origin, scale)
    want, amount = rope(x.reshape(-1, c), heads, d, pairs, at, 10000.0, interleaved, shared, scale)
    # a float64 angle of a far position is itself off: 2^-52 of it
    far = np.abs(at).max() * 2.0 * 2.0 ** -52 * (2.0 if given else 0.0)
    bound = rope_bound(want, amount, dtype) + amount * far
    xt, xd = device(x, dtype)
    yt, yd = empty(n, h, w, c, dtype, (c + 7) // 8 * 8 + 16)
    positions = torch.from_numpy(at.astype(np.int32)).cuda() if given else None
    plan.forward(xd, yd, positions)
    inside(yt[..., :c].reshape(-1, c), want, bound, "rope")
    c8 = (c + 7) // 8 * 8
    assert bool((yt[..., c:c8] == 0).all()) and bool((yt[..., c8:] == 7).all())
    assert torch.equal(yt.view(-1, yt.shape[-1])[:, heads * d:c], xt.view(-1, xt.shape[-1])[:, heads * d:c])
    # in place: the same bits, and what passes is not touched
    zt, zd = device(x, dtype, c8 + 8, fill=7.0)
    plan.forward(zd, zd, positions)
    assert torch.equal(zt[..., :c], yt[..., :c]) and bool((zt[..., c8:] == 7).all())


def test_rope_behind_32_bits():
    """A tensor of more than 2^31 elements: its last tokens."""
    n, side, c = 24, 304, 1024
    x = torch.zeros((n, side, side, c), dtype=torch.bfloat16, device="cuda")
    assert x.numel() > 2 ** 31
    last = torch.randn((side, c), device="cuda").to(torch.bfloat16)
    x[-1, -1] = last
    xd = dn.as_tensor(x, dn.NHWC)
    dn.RopePlan(64, 16, (8, 12, 12), frames=n).forward(xd, xd)
    at = np.stack([np.full(side, n - 1), np.full(side, side - 1), np.arange(side)], -1)
    want, amount = rope(last.double().cpu().numpy(), 16, 64, (8, 12, 12), at)
    inside(x[-1, -1], want, rope_bound(want, amount, "bf16"), "last row")
    assert bool((x[0, 0] == 0).all())


# ------------------------------------------------------------------ norm
NORMS = [(1, 1, 1, 1024), (2, 3, 5, 255), (1, 1, 7, 1), (3, 2, 2, 8), (2, 7, 1, 100), (1, 13, 13, 512), (1, 2, 3, 1500), (1, 1, 5, 4096), (1, 1, 3, 7777), (1, 1, 2, 16384)]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("shape", NORMS)
@pytest.mark.parametrize("outputs", ["y", "sum+y", "sum+y+q", "q32", "q64", "q128", "plain"])
def test_norm(shape, dtype, outputs):
    n, h, w, c = shape
    g = rng(c)
    x, r = held(g.standard_normal(shape) * 3, dtype), held(g.standard_normal(shape), dtype)
    gain = g.standard_normal(c).astype(np.float32)
    plain, with_q, group = outputs == "plain", "q" in outputs, int(outputs[1:]) if outputs[0] == "q" else 0
    s, y = norm(x, None if plain else r, None if plain else gain.astype(np.float64), 1e-3)
    xt, xd = device(x, dtype)
    rt, rd = device(r, dtype, (c + 7) // 8 * 8 + 8, fill=7.0)
    st, sd = empty(n, h, w, c, dtype)
    yt, yd = empty(n, h, w, c, dtype, (c + 7) // 8 * 8 + 8)
    c8 = (c + 7) // 8 * 8
    q = torch.full((n, h, w, c8 + 8), 0x11, dtype=torch.uint8, device="cuda") if with_q else None
    scales = torch.full((n, h, w, -(-c // group) if group else 1), -1.0, device="cuda") if with_q else None
    dn.rmsnorm(xd, yd if "y" in outputs or plain else None, None if plain else torch.from_numpy(gain).cuda(), 1e-3, None if plain else rd,
               sd if "sum" in outputs else None, q, scales, group)
    e = norm_error(c)
    if "sum" in outputs:
        inside(st[..., :c], s, np.abs(s) * (HALF[dtype] + 2.0 ** -24))
        assert bool((st[..., c:] == 0).all())
    if "y" in outputs or plain:
        inside(yt[..., :c], y, np.abs(y) * (HALF[dtype] + e))
        assert bool((yt[..., c:c8] == 0).all()) and bool((yt[..., c8:] == 7).all())
    if with_q:
        step = group or c
        for k in range(scales.shape[-1]):
            part = y[..., k * step:(k + 1) * step]
            scale = np.maximum(np.abs(part).max(-1) / 448, 2.0 ** -126)
            got = scales[..., k].double().cpu().numpy()
            assert (np.abs(got - scale) <= scale * (e + 2.0 ** -23)).all()
            values = q[..., k * step:min(c, (k + 1) * step)].contiguous().view(torch.float8_e4m3fn).double().cpu().numpy() * got[..., None]
            # half a step of e4m3 (2^-4 of the value, 2^-10 scales below its smallest normal), of a value that the norm's error has moved
            inside(values, part, np.abs(part) * (2.0 ** -4 + 2 * e) + got[..., None] * 2.0 ** -10)
        assert bool((q[..., c:c8] == 0).all()) and bool((q[..., c8:] == 0x11).all())


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_norm_in_place_and_without_numbers(dtype):
    """The residual stream updated where it lies; tokens of zeros, of the type's smallest numbers, with an infinity, with a NaN."""
    x = held(rng(5).standard_normal((1, 2, 3, 200)), dtype)
    r = held(rng(6).standard_normal((1, 2, 3, 200)), dtype)
    x[0, 0, 1], r[0, 0, 1] = 0, 0
    x[0, 0, 2], r[0, 0, 2] = held(np.float32(1e-38), dtype), 0
    x[0, 1, 0, 17], r[0, 1, 1, 30] = np.inf, np.nan
    xt, xd = device(x, dtype)
    rt, rd = device(r, dtype)
    q, scales = torch.zeros((1, 2, 3, 200), dtype=torch.float8_e4m3fn, device="cuda"), torch.zeros((1, 2, 3, 4), device="cuda")
    dn.rmsnorm(xd, xd, None, 1e-6, rd, rd, q, scales, 64)         # y over x, the sum over the residual
    s = x + r
    for at in [(0, 0, 0), (0, 0, 1), (0, 0, 2), (0, 1, 2)]:
        want, y = norm(x[at], r[at], None, 1e-6)
        inside(rt[at], want, np.abs(want) * (HALF[dtype] + 2.0 ** -24) + 2.0 ** -149)
        inside(xt[at], y, np.abs(y) * (HALF[dtype] + norm_error(200)) + 2.0 ** -126)
    assert bool((q[0, 0, 1].float() == 0).all()) and bool((scales[0, 0, 1] == 2.0 ** -126).all())
    inf, nan = xt[0, 1, 0].float().cpu().numpy(), xt[0, 1, 1].float().cpu().numpy()
    assert np.isnan(inf[17]) and (np.delete(inf, 17) == 0).all() and np.isnan(nan).all()      # 1 / infinity is 0, and 0 times infinity no number
    assert np.isposinf(rt[0, 1, 0, 17].item()) and np.isnan(rt[0, 1, 1, 30].item()) and int(torch.isnan(rt).sum()) == 1
    assert bool(torch.isnan(scales[0, 1, 1]).all()) and bool(torch.isnan(q[0, 1, 1].float()).all())
    assert bool(torch.isnan(scales[0, 1, 0, 0])) and not bool(torch.isnan(scales[0, 1, 0, 1:]).any())


# ------------------------------------------------------------------ cross attention
def attend(dtype, n, lq, kh, kw, heads, kv_heads, d, kn=None, lengths=None, mask=None, scale=0.0, hidden=None, pitches=(0, 0, 0, 0), seed=1, spread=1.0):
    """One call on seeded inputs against 64 bits; returns the plan and what was compared."""
    g = rng(seed + 7 * lq + kh * kw + d)
    lk, kn = kh * kw, kn or n
    q = held(g.standard_normal((n, 1, lq, heads * d)) * 1.5 * spread, dtype)
    k, v = (held(g.standard_normal((kn, kh, kw, kv_heads * d)), dtype) for _ in range(2))
    allowed = np.ones((n, lq, lk), bool)
    if mask is not None:
        allowed &= np.broadcast_to(mask, allowed.shape)
    if lengths is not None:
        allowed &= np.arange(lk) < np.asarray(lengths)[:, None, None]
    kh_, vh_ = k.copy(), v.copy()
    if hidden is not None:                                       # what no query of an image sees
        assert kn == n
        gone = ~allowed.any(1)
        kh_.reshape(n, lk, -1)[gone], vh_.reshape(n, lk, -1)[gone] = hidden, hidden
    c = heads * d
    qt, qd = device(q, dtype, c + pitches[0], 7.0)
    kt, kd = device(kh_, dtype, kv_heads * d + pitches[1], np.nan)
    vt, vd = device(vh_, dtype, kv_heads * d + pitches[2], np.nan)
    yt, yd = empty(n, 1, lq, c, dtype, c + pitches[3])
    plan = dn.CrossAttentionPlan(heads, kv_heads, d, scale)
    lt = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")
    mt = None if mask is None else torch.from_numpy(mask).cuda().expand(n, lq, lk)
    plan.forward(qd, kd, vd, yd, lt, mt)
    torch.cuda.synchronize()
    plan.check_status()
    want, amount, size = attention(q.reshape(n, lq, c), k.reshape(kn, lk, -1), v.reshape(kn, lk, -1), heads, kv_heads, allowed, scale)
    inside(yt[..., :c].reshape(n, lq, c), want, attention_bound(want, amount, size, d, lk, dtype) + 1e-30, plan.kernel)
    assert bool((yt[..., c:] == 7).all())
    nothing = ~allowed.any(-1)
    assert bool((yt[..., :c].reshape(n, lq, c)[torch.from_numpy(nothing).cuda()] == 0).all())
    return plan, (qt, kt, vt, yt)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("lq", [1, 2, 5, 17, 127, 128, 129, 300])
@pytest.mark.parametrize("keys", [(1, 1), (3, 5), (1, 127), (8, 16), (3, 43), (16, 16), (19, 19), (17, 59)])
def test_attention_lengths_of_queries_and_keys(dtype, lq, keys):
    attend(dtype, 2, lq, *keys, 4, 2, 64)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("d", [8, 16, 24, 32, 40, 56, 64, 72, 80, 96, 104, 120, 128])
@pytest.mark.parametrize("lq", [1, 37])
def test_attention_head_sizes(dtype, d, lq):
    attend(dtype, 1, lq, 7, 41, 2, 1, d)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (3, 3), (6, 2), (5, 1), (16, 4), (7, 7), (24, 3), (16, 1), (40, 2), (160, 1)])
@pytest.mark.parametrize("lq", [1, 3, 70])
def test_attention_head_layouts(dtype, heads, kv_heads, lq):
    attend(dtype, 2, lq, 9, 37, heads, kv_heads, 32)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("d,lq,heads,kv_heads", [(64, 1, 4, 4), (128, 1, 8, 2), (64, 200, 2, 2), (128, 150, 2, 1), (40, 33, 6, 2)])
@pytest.mark.parametrize("hidden", [0.0, np.nan, np.inf, -np.inf])
def test_attention_lengths(dtype, d, lq, heads, kv_heads, hidden):
    """Images of other sizes: nothing, one key, inside and at the end of a tile, all, more than all, below zero; what lies behind is not used."""
    attend(dtype, 9, lq, 20, 25, heads, kv_heads, d, lengths=[0, 1, 127, 128, 129, 300, 500, 100000, -5], hidden=hidden)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("d,lq,heads,kv_heads", [(64, 1, 4, 4), (128, 1, 8, 2), (64, 200, 2, 2), (128, 150, 2, 1), (40, 33, 6, 2)])
@pytest.mark.parametrize("hidden", [None, np.nan, np.inf])
@pytest.mark.parametrize("share", [0.003, 0.5, 0.99])
def test_attention_mask_of_keys(dtype, d, lq, heads, kv_heads, hidden, share):
    mask = rng(int(share * 100)).random((4, 1, 500)) < share
    mask[1] = False                                               # an image that shows nothing
    mask[2, :, :] = False
    mask[2, :, 499] = True                                        # ... or its last key alone
    attend(dtype, 4, lq, 20, 25, heads, kv_heads, d, mask=mask, hidden=hidden)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("d,lq,heads,kv_heads", [(64, 1, 4, 4), (128, 1, 8, 2), (64, 200, 2, 2), (128, 150, 2, 1), (40, 33, 6, 2), (64, 5, 16, 1)])
@pytest.mark.parametrize("share", [0.003, 0.5])
def test_attention_mask_of_each_query(dtype, d, lq, heads, kv_heads, share):
    mask = rng(3).random((3, lq, 517)) < share
    mask[0, 0] = False
    mask[1, lq - 1] = False
    mask[2, :, :256] = False                                      # whole tiles that nobody sees
    attend(dtype, 3, lq, 11, 47, heads, kv_heads, d, mask=mask, lengths=[517, 400, 517])
    attend(dtype, 3, lq, 11, 47, heads, kv_heads, d, mask=mask[:1])     # one image's mask for all: an image stride of zero


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("lq", [1, 150])
def test_attention_of_many_images_to_one_set_of_states(dtype, lq):
    attend(dtype, 5, lq, 13, 13, 4, 2, 64, kn=1, lengths=[169, 3, 0, 50, 128])


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("lq", [1, 140])
def test_attention_channel_ranges_of_wider_tensors(dtype, lq):
    attend(dtype, 2, lq, 13, 17, 4, 2, 64, pitches=(64, 8, 24, 40))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("lq", [1, 140])
@pytest.mark.parametrize("scale", [0.02, -0.3])
def test_attention_scales(dtype, lq, scale):
    attend(dtype, 2, lq, 13, 17, 4, 2, 64, scale=scale)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("lq", [1, 140])
def test_attention_scores_that_grow_with_the_keys(dtype, lq):
    """The largest score moves with nearly every key, by more than what a float's exponent holds in all: the running maximum is what
    counts.  Exact in both: the keys are multiples of one direction."""
    n, heads, d, lk = 1, 2, 64, 700
    q, k = np.zeros((n, 1, lq, heads * d)), np.zeros((n, 1, lk, heads * d))
    q[..., 0::d], k[0, 0, :, 0::d] = 8.0, np.linspace(0, 254, 128).round().repeat(6)[:lk, None]
    k[..., lk // 2:, :] -= 200.0 * (np.arange(heads * d) % d == 0)
    q, k = held(q, dtype), held(k, dtype)
    v = held(rng(4).standard_normal((n, 1, lk, heads * d)), dtype)
    (qt, qd), (kt, kd), (vt, vd) = device(q, dtype), device(k, dtype), device(v, dtype)
    yt, yd = empty(n, 1, lq, heads * d, dtype)
    plan = dn.CrossAttentionPlan(heads, heads, d, 0.5)
    plan.forward(qd, kd, vd, yd)
    want, amount, size = attention(q[:, 0], k[:, 0], v[:, 0], heads, heads, np.ones((n, lq, lk), bool), 0.5)
    inside(yt[:, 0], want, attention_bound(want, amount, size, d, lk, dtype), plan.kernel)


@pytest.mark.parametrize("lq", [1, 40])
def test_attention_behind_32_bits(lq):
    """Keys and values of more than 2^31 elements: the last images."""
    n, side, c, d = 400, 76, 1024, 128
    k = torch.zeros((n, side, side, c), dtype=torch.bfloat16, device="cuda")
    v = torch.zeros_like(k)
    assert k.numel() > 2 ** 31
    q = torch.randn((n, 1, lq, c), device="cuda").to(torch.bfloat16)
    k[-1], v[-1] = torch.randn((2, side, side, c), device="cuda").to(torch.bfloat16)
    yt, yd = empty(n, 1, lq, c, "bf16")
    plan = dn.CrossAttentionPlan(8, 8, d)
    plan.forward(dn.as_tensor(q, dn.NHWC), dn.as_tensor(k, dn.NHWC), dn.as_tensor(v, dn.NHWC), yd)
    plan.check_status()
    f = lambda t: t[-1:].double().cpu().numpy().reshape(1, -1, c)  # noqa: E731
    want, amount, size = attention(f(q), f(k), f(v), 8, 8, np.ones((1, lq, side * side), bool))
    inside(yt[-1:, 0], want, attention_bound(want, amount, size, d, side * side, "bf16"), plan.kernel)
    assert bool((yt[:-1] == 0).all())


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("lq,heads,kv_heads", [(1, 8, 8), (1, 16, 2), (30, 4, 4), (300, 4, 2)])
def test_attention_gives_the_same_bits_every_time(dtype, lq, heads, kv_heads):
    plan, (qt, kt, vt, yt) = attend(dtype, 2, lq, 38, 38, heads, kv_heads, 64)
    first = yt.clone()
    for _ in range(3):
        yt.fill_(3.0)
        plan.forward(*(dn.as_tensor(t, dn.NHWC) for t in (qt, kt, vt, yt)))
        assert torch.equal(first, yt)


# ------------------------------------------------------------------ the block
def block(dtype, side, channels, heads, kv_heads, lq, n, seed):
    """A cross-attention block: queries are normed and projected, the map is projected, both turn with their positions, attention, the
    projection back, and the norm of the residual's sum.  Returns the buffers, a function that runs it, and the plans."""
    g = rng(seed)
    d = channels // heads
    mode = dn.MODE_BF16 if dtype == "bf16" else dn.MODE_FP32
    b = {}
    for name, shape in dict(x=(n, 1, lq, channels), states=(n, side, side, channels)).items():
        b[name] = device(held(g.standard_normal(shape), dtype), dtype)
    for name, shape in dict(normed=(n, 1, lq, channels), q=(n, 1, lq, channels), qr=(n, 1, lq, channels), kv=(n, side, side, 2 * kv_heads * d), o=(n, 1, lq, channels),
                            p=(n, 1, lq, channels), total=(n, 1, lq, channels), y=(n, 1, lq, channels)).items():
        b[name] = empty(*shape, dtype)
    b["at"] = torch.from_numpy(g.integers(0, 2000, (n * lq, 3)).astype(np.int32)).cuda()
    b["gain"] = torch.from_numpy(g.standard_normal(channels).astype(np.float32)).cuda()
    b["e4m3"] = torch.zeros((n, 1, lq, channels), dtype=torch.float8_e4m3fn, device="cuda")
    b["scales"] = torch.zeros((n, 1, lq, channels // 64), device="cuda")

    def projection(c, n_out, h, w):
        plan = dn.ConvPlan(n, c, h, w, n_out, 1, mode=mode)
        weights, biases = g.standard_normal((n_out, c, 1, 1)).astype(np.float32) / np.sqrt(c).astype(np.float32), g.standard_normal(n_out).astype(np.float32)
        plan.set_params(weights, biases)
        plan.w = weights.reshape(n_out, c).astype(np.float64), biases.astype(np.float64)
        return plan

    pq, pkv, po = projection(channels, channels, 1, lq), projection(channels, 2 * kv_heads * d, side, side), projection(channels, channels, 1, lq)
    rq, rk = dn.RopePlan(d, heads, (d // 8, d // 8, d // 8)), dn.RopePlan(d, kv_heads, (0, d // 4, d // 4))
    attention_plan = dn.CrossAttentionPlan(heads, kv_heads, d)
    kv, ck = b["kv"][0], kv_heads * d
    es = kv.element_size()
    dt = dn.BF16 if dtype == "bf16" else dn.F32
    b["k"] = kv, dn.Tensor(kv.data_ptr(), dn.NHWC, dt, n, ck, side, side, 2 * ck)
    b["v"] = kv, dn.Tensor(kv.data_ptr() + ck * es, dn.NHWC, dt, n, ck, side, side, 2 * ck)

    def run():
        D = {name: t[1] for name, t in b.items() if isinstance(t, tuple)}
        dn.rmsnorm(D["x"], D["normed"], b["gain"])
        pq.forward(D["normed"], D["q"])
        pkv.forward(D["states"], D["kv"])
        rq.forward(D["q"], D["qr"], b["at"])
        rk.forward(D["k"], D["k"])                                # in place: the keys' half of the tensor
        attention_plan.forward(D["qr"], D["k"], D["v"], D["o"])
        po.forward(D["o"], D["p"])
        dn.rmsnorm(D["p"], D["y"], b["gain"], residual=D["x"], total=D["total"], e4m3=b["e4m3"], scales=b["scales"], group=64)

    return b, run, (pq, pkv, po, rq, rk, attention_plan)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("lq", [1, 45])
def test_a_block_step_by_step(dtype, lq):
    """Every step of the block against 64 bits on what the step before left."""
    n, side, channels, heads, kv_heads = 2, 13, 256, 4, 2
    d, ck = channels // heads, channels // heads * kv_heads
    b, run, (pq, pkv, po, rq, rk, plan) = block(dtype, side, channels, heads, kv_heads, lq, n, 20 + lq)
    run()
    torch.cuda.synchronize()
    plan.check_status()
    f = {name: t[0].double().cpu().numpy().reshape(n * t[0].shape[1] * t[0].shape[2], -1) for name, t in b.items() if isinstance(t, tuple)}
    gain = b["gain"].double().cpu().numpy()
    _, want = norm(f["x"], None, gain, 1e-6)
    inside(f["normed"], want, np.abs(want) * (HALF[dtype] + norm_error(channels)), "norm")

    def projected(x, p, got, label):
        weights = held(p.w[0], dtype)
        want, amount = x @ weights.T + p.w[1], np.abs(x) @ np.abs(weights).T + np.abs(p.w[1])
        inside(got, want, np.abs(want) * HALF[dtype] + amount * channels * 2.0 ** -24, label)

    projected(f["normed"], pq, f["q"], "query projection")
    want, amount = rope(f["q"], heads, d, (d // 8,) * 3, b["at"].cpu().numpy())
    inside(f["qr"], want, rope_bound(want, amount, dtype) + amount * 2000 * 2.0 ** -52, "query positions")
    weights, biases = held(pkv.w[0], dtype), pkv.w[1]
    kv, size = f["states"] @ weights.T + biases, np.abs(f["states"]) @ np.abs(weights).T + np.abs(biases)
    off = np.abs(kv) * HALF[dtype] + size * channels * 2.0 ** -24
    inside(f["kv"][:, ck:], kv[:, ck:], off[:, ck:], "values")
    want, amount = rope(kv[:, :ck], kv_heads, d, (0, d // 4, d // 4), grid_positions(n, side, side))
    _, both = rope(off[:, :ck], kv_heads, d, (0, d // 4, d // 4), grid_positions(n, side, side))
    inside(f["kv"][:, :ck], want, rope_bound(want, amount, dtype) + both * 1.01, "keys")
    seen = np.ones((n, lq, side * side), bool)
    want, amount, size = attention(f["qr"].reshape(n, lq, -1), f["kv"][:, :ck].reshape(n, -1, ck), f["kv"][:, ck:].reshape(n, -1, ck), heads, kv_heads, seen)
    inside(f["o"].reshape(n, lq, -1), want, attention_bound(want, amount, size, d, side * side, dtype), "attention")
    projected(f["o"], po, f["p"], "projection back")
    s, y = norm(f["p"], f["x"], gain, 1e-6)
    inside(f["total"], s, np.abs(s) * (HALF[dtype] + 2.0 ** -24), "sum")
    inside(f["y"], y, np.abs(y) * (HALF[dtype] + norm_error(channels)), "output")
    scales = b["scales"].double().cpu().numpy().reshape(n * lq, -1).repeat(64, 1)
    inside(b["e4m3"].double().cpu().numpy().reshape(n * lq, -1) * scales, y, np.abs(y) * (2.0 ** -4 + 2 * norm_error(channels)) + scales * 2.0 ** -10, "output in 8 bits")


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("lq", [1, 45])
def test_a_block_captured_and_on_another_stream(dtype, lq):
    b, run, plans = block(dtype, 13, 256, 4, 2, lq, 2, 31)
    run()
    torch.cuda.synchronize()
    outputs = [b[k][0] for k in ("total", "y")] + [b["e4m3"].view(torch.uint8), b["scales"]]
    want = [t.clone() for t in outputs]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for t in outputs:
            t.zero_()
        run()
    side.synchronize()
    assert all(torch.equal(a, w) for a, w in zip(outputs, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        run()
    fresh = torch.randn_like(b["x"][0].float()).to(b["x"][0].dtype)
    for x in (b["x"][0].clone(), fresh):
        b["x"][0].copy_(x)
        run()
        torch.cuda.synchronize()
        want = [t.clone() for t in outputs]
        for t in outputs:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, w) for a, w in zip(outputs, want))
    plans[-1].check_status()


def test_attention_calls_at_once_on_two_streams():
    """One plan, two streams, calls of different sizes that overlap."""
    plan, jobs = dn.CrossAttentionPlan(8, 2, 64), []
    for i, (n, lq, side) in enumerate([(2, 1, 38), (3, 200, 38), (1, 1, 76), (2, 64, 19)]):
        g = torch.Generator(device="cuda").manual_seed(i)
        q = torch.randn((n, 1, lq, 512), generator=g, device="cuda").to(torch.bfloat16)
        k, v = torch.randn((2, n, side, side, 128), generator=g, device="cuda").to(torch.bfloat16)
        ys = [torch.zeros_like(q) for _ in range(2)]
        jobs.append((q, k, v, ys))
    D = lambda t: dn.as_tensor(t, dn.NHWC)  # noqa: E731
    for q, k, v, ys in jobs:
        plan.forward(D(q), D(k), D(v), D(ys[0]))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(10):
        for i, (q, k, v, ys) in enumerate(jobs):
            with torch.cuda.stream(streams[i % 2]):
                plan.forward(D(q), D(k), D(v), D(ys[1]))
    torch.cuda.synchronize()
    plan.check_status()
    assert all(torch.equal(ys[0], ys[1]) for _, _, _, ys in jobs)
