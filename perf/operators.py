"""The parts of a cross-attention block over channels-last feature maps, as cases that can be timed.

Three operators, each in its plain form (elementary torch operations in 32 bits) and as a call of the framework:

* ``rope``: rotary positions with the axes time, row and column, of a map, a clip of maps, or tokens with given positions;
* ``attention``: attention of query tokens (one token, a set of queries, another map) to a feature map's states;
* ``norm``: root-mean-square norm with the residual's addition, in the tensors' own type and as e4m3 with scales.

Maps are those of the benchmark's networks: 608/32 = 19, 38 and 76 pixels a side, 255, 512 and 1024 channels, batches
of 1 to 32; the other sizes are odd on purpose.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


# ---------------------------------------------------------------------------------------------------- the cases
def _rope(name, dtype, n, h, w, c, heads, head_dim, t, y, x, frames, interleaved, shared, given):
    return {"name": name, "op": "rope", "dtype": dtype, "n": n, "h": h, "w": w, "c": c, "heads": heads, "head_dim": head_dim, "pairs_t": t, "pairs_y": y,
            "pairs_x": x, "frames": frames, "interleaved": interleaved, "shared": shared, "given": given}


def _norm(name, dtype, n, h, w, c, total, y, e4m3, group):
    return {"name": name, "op": "norm", "dtype": dtype, "n": n, "h": h, "w": w, "c": c, "sum": total, "y": y, "e4m3": e4m3, "group": group}


def _attention(name, dtype, n, lq, kh, kw, heads, kv_heads, head_dim, lengths, mask):
    return {"name": name, "op": "attention", "dtype": dtype, "n": n, "lq": lq, "kh": kh, "kw": kw, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim,
            "lengths": lengths, "mask": mask}


def listed():
    return [
        # one generated token's queries, keys and values in one tensor; queries and keys turn, its position is a triple
        _rope("rope token bf16", "bf16", 1, 1, 1, 1536, 20, 64, 8, 12, 12, 1, False, True, True),
        # maps of an odd size and head, neighbouring channels as pairs, rows and columns with spectra of their own, channels left over
        _rope("rope map f32 odd", "f32", 3, 19, 25, 511, 7, 72, 0, 18, 18, 1, True, False, False),
        # a clip of sixteen frames on the finest map of the 608-pixel detector
        _rope("rope clip bf16", "bf16", 16, 76, 76, 1024, 16, 64, 8, 12, 12, 16, False, True, False),
        # one token's residual and norm
        _norm("norm token bf16", "bf16", 1, 1, 1, 1024, True, True, False, 0),
        # the detector's head channels, whose number is odd, in full precision
        _norm("norm map f32 odd", "f32", 8, 19, 19, 255, True, True, False, 0),
        # a batch of fine maps whose next product takes 8 bits with a scale for 128 channels each
        _norm("norm map e4m3", "bf16", 16, 76, 76, 512, True, False, True, 128),
        # one token attends to the coarsest map of one image: latency
        _attention("attend token bf16", "bf16", 1, 1, 19, 19, 8, 8, 64, False, False),
        # a batch of tokens, query heads that share keys, images of other sizes in one padded batch: memory
        _attention("attend tokens batch", "bf16", 32, 1, 76, 76, 16, 4, 128, True, False),
        # a hundred detection queries in full precision
        _attention("attend queries f32", "f32", 8, 100, 38, 38, 8, 8, 32, False, False),
        # queries that look into their own boxes (some of them empty), odd sizes throughout
        _attention("attend boxes odd", "bf16", 3, 37, 17, 59, 12, 4, 40, True, True),
        # a coarser map's pixels attend to the finest map
        _attention("attend map d64", "bf16", 8, 1444, 76, 76, 8, 8, 64, False, False),
        # the finest map to the finest map of another view
        _attention("attend map d128", "bf16", 8, 5776, 76, 76, 8, 8, 128, False, False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    dtype = rng.choice(["bf16", "bf16", "f32"])
    op = rng.choice(["rope", "norm", "attention", "attention"])
    if op == "rope":
        head_dim = 8 * rng.randint(2, 16)
        pairs = head_dim // 2 - rng.choice([0, 0, rng.randint(0, head_dim // 4)])
        t = rng.choice([0, pairs // 4])
        y = (pairs - t) // 2
        heads = _log(rng, 1, 24)
        h, w, n = _log(rng, 1, 76), _log(rng, 1, 76), _log(rng, 1, 16)
        c = heads * head_dim + rng.choice([0, rng.randint(1, 300)])
        while n * h * w * c > 16 * 5776 * 1024:
            n, h = max(1, n // 2), max(1, h - h // 4)
        frames = rng.choice([f for f in (1, 2, 4, 8, 16) if n % f == 0])
        case = _rope("", dtype, n, h, w, c, heads, head_dim, t, y, pairs - t - y, frames, rng.random() < 0.5, rng.random() < 0.5, rng.random() < 0.4)
    elif op == "norm":
        c, h, w, n = _log(rng, 8, 4096), _log(rng, 1, 76), _log(rng, 1, 76), _log(rng, 1, 32)
        while n * h * w * c > 16 * 5776 * 512:
            n, h = max(1, n // 2), max(1, h - h // 4)
        e4m3 = rng.random() < 0.5
        case = _norm("", dtype, n, h, w, c, rng.random() < 0.6, not e4m3 or rng.random() < 0.3, e4m3, rng.choice([0, 32, 64, 128]))
    else:
        head_dim = 8 * rng.randint(2, 16)
        kv_heads, group = _log(rng, 1, 16), rng.choice([1, 1, 2, 3, 4, 8])
        heads, n = kv_heads * group, _log(rng, 1, 32)
        lq = rng.choice([1, _log(rng, 1, 300), _log(rng, 64, 5776)])
        kh, kw = _log(rng, 1, 76), _log(rng, 1, 76)
        most = 8 * 8 * 5776 * 5776 * (1 if dtype == "bf16" else 0.1)  # scores; a full-precision one costs about ten times as much
        while n * heads * lq * kh * kw > most or n * kh * kw * kv_heads * head_dim > 32 * 5776 * 512:
            n, lq = max(1, n // 2), max(1, lq - lq // 4)
        mask = lq * kh * kw * n < 1 << 28 and rng.random() < 0.3
        case = _attention("", dtype, n, lq, kh, kw, heads, kv_heads, head_dim, rng.random() < 0.4, mask)
    del case["name"]
    return case


# ---------------------------------------------------------------------------------------------------- inputs
def _pitch(c):
    return (c + 7) // 8 * 8


def _map(g, n, h, w, c, dtype, scale=1.0):
    """A channels-last map [n, h, w, pitch] whose padding channels are zero."""
    t = torch.randn((n, h, w, _pitch(c)), generator=g, device="cuda", dtype=torch.float32).mul_(scale)
    t[..., c:] = 0
    return t.to(dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype, s = DTYPES[case["dtype"]], {"case": case}
    if case["op"] == "rope":
        n, h, w, c = (case[k] for k in ("n", "h", "w", "c"))
        s["x"] = _map(g, n, h, w, c, dtype)
        s["positions"] = torch.randint(0, 100000, (n * h * w, 3), generator=g, device="cuda", dtype=torch.int32) if case["given"] else None
    elif case["op"] == "norm":
        n, h, w, c = (case[k] for k in ("n", "h", "w", "c"))
        s["x"], s["residual"] = _map(g, n, h, w, c, dtype), _map(g, n, h, w, c, dtype, 2.0)
        s["gain"] = torch.randn(c, generator=g, device="cuda").mul_(0.2).add_(1.0)
    else:
        n, lq, kh, kw, d = (case[k] for k in ("n", "lq", "kh", "kw", "head_dim"))
        s["q"] = _map(g, n, 1, lq, case["heads"] * d, dtype, 1.5)
        s["k"] = _map(g, n, kh, kw, case["kv_heads"] * d, dtype)
        s["v"] = _map(g, n, kh, kw, case["kv_heads"] * d, dtype)
        # images of other sizes padded to the largest: from a quarter of it up, the first one whole
        s["lengths"] = None
        if case["lengths"]:
            s["lengths"] = torch.randint(max(1, kh * kw // 4), kh * kw + 1, (n,), generator=g, device="cuda", dtype=torch.int32)
            s["lengths"][0] = kh * kw
        s["mask"] = None
        if case["mask"]:  # every query its box of the map; a box may be empty
            lo = torch.rand((n, lq, 2), generator=g, device="cuda")
            hi = lo + torch.rand((n, lq, 2), generator=g, device="cuda") * 0.7 - 0.05
            ys, xs = (torch.arange(kh, device="cuda") + 0.5) / kh, (torch.arange(kw, device="cuda") + 0.5) / kw
            rows, columns = (ys >= lo[..., :1]) & (ys < hi[..., :1]), (xs >= lo[..., 1:]) & (xs < hi[..., 1:])
            s["mask"] = (rows[..., :, None] & columns[..., None, :]).reshape(n, lq, kh * kw)
    if own:
        _handles(s)
    return s


def _handles(s):
    """The plans, output buffers and descriptors that a program keeps beside its tensors."""
    import darknet_b200 as dn
    case = s["case"]
    nhwc = lambda t, c: dn.as_tensor(t, dn.NHWC, c)  # noqa: E731
    if case["op"] == "rope":
        s["plan"] = dn.RopePlan(case["head_dim"], case["heads"], (case["pairs_t"], case["pairs_y"], case["pairs_x"]), frames=case["frames"],
                                interleaved=case["interleaved"], shared=case["shared"])
        s["y"] = torch.zeros_like(s["x"])
        s["tensors"] = nhwc(s["x"], case["c"]), nhwc(s["y"], case["c"])
    elif case["op"] == "norm":
        n, h, w, c = (case[k] for k in ("n", "h", "w", "c"))
        s["total"] = torch.zeros_like(s["x"]) if case["sum"] else None
        s["y"] = torch.zeros_like(s["x"]) if case["y"] else None
        s["q"] = torch.zeros(s["x"].shape, device="cuda", dtype=torch.float8_e4m3fn) if case["e4m3"] else None
        s["scales"] = torch.zeros((n, h, w, _groups(case)), device="cuda") if case["e4m3"] else None
        s["tensors"] = [None if t is None else nhwc(t, c) for t in (s["x"], s["residual"], s["total"], s["y"])]
    else:
        s["plan"] = dn.CrossAttentionPlan(case["heads"], case["kv_heads"], case["head_dim"])
        s["y"] = torch.zeros_like(s["q"])
        cq, ck = case["heads"] * case["head_dim"], case["kv_heads"] * case["head_dim"]
        s["tensors"] = nhwc(s["q"], cq), nhwc(s["k"], ck), nhwc(s["v"], ck), nhwc(s["y"], cq)


def _groups(case):
    return -(-case["c"] // case["group"]) if case["group"] else 1


# ---------------------------------------------------------------------------------------------------- one pass
def run(state):
    if own:
        return _run_own(state)
    return {"rope": _plain_rope, "norm": _plain_norm, "attention": _plain_attention}[state["case"]["op"]](state)


def _run_own(s):
    case = s["case"]
    if case["op"] == "rope":
        s["plan"].forward(*s["tensors"], positions=s["positions"])
        return {"y": s["y"]}
    if case["op"] == "norm":
        import darknet_b200 as dn
        x, residual, total, y = s["tensors"]
        dn.rmsnorm(x, y, s["gain"], residual=residual, total=total, e4m3=s["q"], scales=s["scales"], group=case["group"])
        return {"sum": s["total"], "y": s["y"], "e4m3": s["q"], "scales": s["scales"]}
    s["plan"].forward(*s["tensors"], lengths=s["lengths"], mask=s["mask"])
    return {"y": s["y"]}


def _plain_rope(s):
    case, x = s["case"], s["x"]
    n, h, w, d, heads = x.shape[0], x.shape[1], x.shape[2], case["head_dim"], case["heads"]
    by_axis = [case["pairs_t"], case["pairs_y"], case["pairs_x"]]
    pairs = sum(by_axis)
    i = torch.arange(pairs, device="cuda", dtype=torch.float64)
    sizes = torch.tensor(by_axis, device="cuda")
    axis = torch.repeat_interleave(torch.arange(3, device="cuda"), sizes, output_size=pairs)
    if case["shared"]:
        power = i / pairs
    else:
        power = (i - (torch.cumsum(sizes, 0) - sizes)[axis]) / sizes[axis]
    frequency = 10000.0 ** -power
    if s["positions"] is None:
        at = torch.stack(torch.meshgrid(torch.arange(n, device="cuda") % case["frames"], torch.arange(h, device="cuda"), torch.arange(w, device="cuda"), indexing="ij"), -1)
    else:
        at = s["positions"].view(n, h, w, 3)
    angle = at[..., axis].double() * frequency                                  # in 64 bits: far positions lose their angle in 32
    cos, sin = angle.cos().float()[..., None, :], angle.sin().float()[..., None, :]
    v = x[..., :heads * d].float().unflatten(-1, (heads, d))
    if case["interleaved"]:
        a, b = v[..., 0:2 * pairs:2], v[..., 1:2 * pairs:2]
        turned = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
    else:
        a, b = v[..., :pairs], v[..., pairs:2 * pairs]
        turned = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
    turned = torch.cat((turned, v[..., 2 * pairs:]), -1).flatten(-2)
    return {"y": torch.cat((turned.to(x.dtype), x[..., heads * d:]), -1)}


def _plain_norm(s):
    case, x = s["case"], s["x"]
    c = case["c"]
    total = x.float() + s["residual"].float()
    y = total[..., :c] * torch.rsqrt(total[..., :c].square().mean(-1, keepdim=True) + 1e-6) * s["gain"]
    out = {"sum": total.to(x.dtype) if case["sum"] else None, "y": None, "e4m3": None, "scales": None}
    y = torch.nn.functional.pad(y, (0, _pitch(c) - c))
    if case["y"]:
        out["y"] = y.to(x.dtype)
    if case["e4m3"]:
        group, groups = case["group"] or _pitch(c), _groups(case)
        parts = torch.nn.functional.pad(y[..., :c], (0, groups * group - c)).unflatten(-1, (groups, group))
        scales = (parts.abs().amax(-1) / 448).clamp_min(2.0 ** -126)
        out["e4m3"] = torch.nn.functional.pad((parts / scales[..., None]).flatten(-2)[..., :c], (0, _pitch(c) - c)).to(torch.float8_e4m3fn)
        out["scales"] = scales
    return out


def _plain_attention(s):
    case, q, k, v = s["case"], s["q"], s["k"], s["v"]
    n, lq, lk, d, kv = case["n"], case["lq"], case["kh"] * case["kw"], case["head_dim"], case["kv_heads"]
    group = case["heads"] // kv
    rows = q.float()[..., :case["heads"] * d].reshape(n, lq, kv, group, d).permute(0, 2, 3, 1, 4).reshape(n, kv, group * lq, d)
    keys = k.float()[..., :kv * d].reshape(n, lk, kv, d).transpose(1, 2)
    values = v.float()[..., :kv * d].reshape(n, lk, kv, d).transpose(1, 2)
    scores = (rows @ keys.transpose(-1, -2)).mul_(d ** -0.5).view(n, kv, group, lq, lk)
    if s["lengths"] is not None:
        scores.masked_fill_((torch.arange(lk, device="cuda") >= s["lengths"][:, None])[:, None, None, None, :], -math.inf)
    if s["mask"] is not None:
        scores.masked_fill_(~s["mask"][:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = scores.sub_(top.masked_fill(top == -math.inf, 0.0)).exp_()
    norm = p.sum(-1, keepdim=True)
    out = (p.view(n, kv, group * lq, lk) @ values).view(n, kv, group, lq, d) / norm.masked_fill(norm == 0, 1.0)  # a row without keys: zero
    out = out.permute(0, 3, 1, 2, 4).reshape(n, 1, lq, case["heads"] * d)
    return {"y": torch.nn.functional.pad(out, (0, q.shape[-1] - out.shape[-1])).to(q.dtype)}


# ---------------------------------------------------------------------------------------------------- what it takes
def work(case):
    size = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "rope":
        tokens = case["n"] * case["h"] * case["w"]
        pairs = case["pairs_t"] + case["pairs_y"] + case["pairs_x"]
        return {"bytes": tokens * (2 * size * case["c"] + (12 if case["given"] else 0)), "flops": 6 * tokens * case["heads"] * pairs}
    if case["op"] == "norm":
        tokens, c = case["n"] * case["h"] * case["w"], case["c"]
        written = size * c * (case["sum"] + case["y"]) + (c + 4 * _groups(case) if case["e4m3"] else 0)
        return {"bytes": tokens * (2 * size * c + written) + 4 * c, "flops": 6 * tokens * c}
    n, lq, lk, d = case["n"], case["lq"], case["kh"] * case["kw"], case["head_dim"]
    keys = lk * (0.625 if case["lengths"] else 1.0)  # lengths are uniform from a quarter of the map up
    moved = 2 * n * lq * case["heads"] * d * size + 2 * n * keys * case["kv_heads"] * d * size + (n * lq * keys if case["mask"] else 0)
    return {"bytes": moved, "flops": 4 * n * case["heads"] * lq * keys * d}


# ---------------------------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rope":
        return _exact_rope(case, s)
    if case["op"] == "norm":
        return _exact_norm(case, s)
    return _exact_attention(case, s)


def _exact_rope(case, s):
    y, d = s["x"].double(), case["head_dim"]
    n, h, w = y.shape[:3]
    given = None if s["positions"] is None else s["positions"].double().view(n, h, w, 3)
    grid = [(torch.arange(n, device="cuda") % case["frames"]).view(n, 1, 1), torch.arange(h, device="cuda").view(1, h, 1), torch.arange(w, device="cuda").view(1, 1, w)]
    counts = [case["pairs_t"], case["pairs_y"], case["pairs_x"]]
    i, pairs = 0, sum(counts)
    for axis in range(3):
        for j in range(counts[axis]):
            f = math.pow(10000.0, -(i / pairs if case["shared"] else j / counts[axis]))
            theta = (grid[axis].double() if given is None else given[..., axis]) * f
            turn = torch.polar(torch.ones_like(theta), theta)[..., None]
            first, second = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + pairs)
            a, b = y[..., first:case["heads"] * d:d], y[..., second:case["heads"] * d:d]
            z = torch.complex(a, b) * turn
            y[..., first:case["heads"] * d:d], y[..., second:case["heads"] * d:d] = z.real, z.imag
            i += 1
    return {"y": y}


def _exact_norm(case, s):
    c = case["c"]
    total = s["x"].double() + s["residual"].double()
    length = torch.linalg.vector_norm(total[..., :c], dim=-1, keepdim=True)
    y = total[..., :c] / torch.sqrt(length * length / c + 1e-6) * s["gain"].double()
    whole = torch.zeros_like(total)
    whole[..., :c] = y
    out = {"sum": total if case["sum"] else None, "y": whole if case["y"] else None, "e4m3": None, "scales": None}
    if case["e4m3"]:
        values, scales = torch.zeros_like(total), []
        step = case["group"] or c
        for at in range(0, c, step):
            scales.append((y[..., at:at + step].abs().max(-1).values / 448).clamp_min(2.0 ** -126))
            values[..., at:min(c, at + step)] = y[..., at:at + step] / scales[-1][..., None]
        out["e4m3"], out["scales"] = values, torch.stack(scales, -1)
    return out


def _exact_attention(case, s):
    n, lq, lk, d = case["n"], case["lq"], case["kh"] * case["kw"], case["head_dim"]
    group = case["heads"] // case["kv_heads"]
    y = torch.zeros(s["q"].shape, device="cuda", dtype=torch.float64)
    for image in range(n):
        allowed = torch.ones((lq, lk), device="cuda", dtype=torch.bool) if s["mask"] is None else s["mask"][image].clone()
        if s["lengths"] is not None:
            allowed &= torch.arange(lk, device="cuda")[None] < s["lengths"][image]
        some = allowed.any(-1)
        for head in range(case["heads"]):
            at, of = slice(head * d, head * d + d), slice(head // group * d, head // group * d + d)
            scores = torch.einsum("id,jd->ij", s["q"][image, 0, :, at].double(), s["k"][image].reshape(lk, -1)[:, of].double()) / math.sqrt(d)
            weights = torch.softmax(torch.where(allowed, scores, -math.inf), -1)
            y[image, 0, :, at] = torch.where(some[:, None], torch.nan_to_num(weights) @ s["v"][image].reshape(lk, -1)[:, of].double(), 0.0)
    return {"y": y}
