"""Plain implementations in 64 bits of the operators around cross attention, with the error that arithmetic in the kernels' types may make."""
import numpy as np

HALF = {"bf16": 2.0 ** -8, "f32": 2.0 ** -24}     # half a step of the type, relative to the value
U = 2.0 ** -24                                     # the same of the kernels' own sums


def rope(x, heads, head_dim, pairs, positions, base=10000.0, interleaved=False, shared=True, scale=(1.0, 1.0, 1.0)):
    """x [tokens, c] in float64, positions [tokens, 3]: the turned tensor, and the sum of what each output is made of."""
    y, amount = x.copy(), np.abs(x)
    p, i = sum(pairs), 0
    for axis in range(3):
        for j in range(pairs[axis]):
            f = float(np.float32(base)) ** -(i / p if shared else j / pairs[axis])
            theta = positions[:, axis].astype(np.float64) * float(np.float32(scale[axis])) * f
            for h in range(heads):
                a = h * head_dim + (2 * i if interleaved else i)
                b = h * head_dim + (2 * i + 1 if interleaved else i + p)
                y[:, a] = x[:, a] * np.cos(theta) - x[:, b] * np.sin(theta)
                y[:, b] = x[:, a] * np.sin(theta) + x[:, b] * np.cos(theta)
                amount[:, a] = amount[:, b] = np.abs(x[:, a]) + np.abs(x[:, b])
            i += 1
    return y, amount


def grid_positions(n, h, w, frames=1, origin=(0, 0, 0)):
    t, y, x = np.meshgrid(np.arange(n) % frames, np.arange(h), np.arange(w), indexing="ij")
    return np.stack([t, y, x], -1).reshape(-1, 3) + np.asarray(origin)


def rope_bound(y, amount, dtype):
    """Half a step of the output; sine and cosine off by the rounding of the turn to 24 bits (2 pi 2^-26) and 2^-21.4 (the worst of a
    fast sine on one turn), and three roundings of the products and their sum."""
    return HALF[dtype] * np.abs(y) + amount * (2 * np.pi * 2.0 ** -26 + 2.0 ** -21.4 + 3 * U)


def norm(x, r, gain, eps):
    s = x if r is None else x + r
    y = s / np.sqrt((s * s).mean(-1, keepdims=True) + float(np.float32(eps)))
    return s, y if gain is None else y * gain


def norm_error(c):
    """Relative error of a norm in fp32: the squares' rounding and their sum (c / 32 terms one after another, then a tree), halved by the
    root; the sum before it, the mean, the root, the quotient and two products."""
    return (c / 32 + 24) * U


def attention(q, k, v, heads, kv_heads, allowed, scale=None):
    """q [n, lq, heads*d], k, v [n or 1, lk, kv_heads*d] in float64, allowed bool [n, lq, lk].  Returns the output, sum p|v|, and the
    largest sum over channels of |q||k| * scale that a row meets."""
    n, lq, _ = q.shape
    d = q.shape[2] // heads
    scale = float(np.float32(scale)) if scale else 1.0 / np.sqrt(d)
    y, amount, size = np.zeros_like(q), np.zeros_like(q), np.zeros_like(q)
    for i in range(n):
        for h in range(heads):
            at, of = slice(h * d, h * d + d), slice(h // (heads // kv_heads) * d, h // (heads // kv_heads) * d + d)
            ki, vi = k[i % k.shape[0] if k.shape[0] > 1 else 0][:, of], v[i if v.shape[0] > 1 else 0][:, of]
            seen = allowed[i]
            some = seen.any(0)                                            # what no query sees is not used
            ki, vi = np.where(some[:, None], ki, 0.0), np.where(some[:, None], vi, 0.0)
            s = np.where(seen, q[i][:, at] @ ki.T * scale, -np.inf)
            top = s.max(-1, keepdims=True)
            p = np.exp(s - np.where(np.isfinite(top), top, 0.0))
            total = p.sum(-1, keepdims=True)
            p = p / np.where(total == 0, 1.0, total)
            y[i][:, at], amount[i][:, at] = p @ vi, p @ np.abs(vi)
            size[i][:, at] = (np.where(seen, np.abs(q[i][:, at]) @ np.abs(ki).T, 0.0).max(-1, keepdims=True)) * abs(scale)
    return y, amount, size


def attention_bound(y, amount, size, d, lk, dtype):
    """Half a step of the output; weights rounded to the type before they meet the values (bf16: half a step each, of the sum of p|v|); a
    weight's relative error from its score's (d + 2 roundings of sum |q||k| scale, twice: its own and the row's largest score's), from the
    exponential (2^-21) and from lk roundings in each of the two sums."""
    weights = HALF["bf16"] if dtype == "bf16" else 0.0
    return HALF[dtype] * np.abs(y) + amount * (weights + 2 * (d + 4) * U * size + 2.0 ** -20 + 2 * lk * U)
