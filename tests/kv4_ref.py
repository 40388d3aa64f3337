"""The 4-bit key / value cache and the attention over it, from their formulas in 64-bit numpy."""
import numpy as np


def rope(positions, rot, theta=10000.0):
    """[positions][rot / 2] of (sin, cos), in f32."""
    freq = theta ** (-np.arange(0, rot, 2, dtype=np.float64) / rot)
    a = np.arange(positions, dtype=np.float64)[:, None] * freq
    return np.stack((np.sin(a), np.cos(a)), -1).astype(np.float32)


def rotate(x, table, pos, rot, neox):
    """x [tokens, heads, dim] turned by the angles of its positions, in 64 bits."""
    x = x.astype(np.float64)
    if not rot:
        return x
    sin, cos = (table[pos].astype(np.float64)[:, None, :, i] for i in (0, 1))
    out = x.copy()
    a, b = (slice(0, rot // 2), slice(rot // 2, rot)) if neox else (slice(0, rot, 2), slice(1, rot, 2))
    with np.errstate(invalid="ignore", over="ignore"):
        out[..., a] = x[..., a] * cos - x[..., b] * sin
        out[..., b] = x[..., b] * cos + x[..., a] * sin if neox else x[..., a] * sin + x[..., b] * cos
    return out


def quantize(x):
    """-> codes [..., dim], step and minimum [..., dim / 32] (64-bit numbers that are half precision)."""
    b = x.reshape(*x.shape[:-1], -1, 32)
    bad = ~np.isfinite(b).all(-1)
    b = np.where(bad[..., None], 0.0, b)
    big = 65504.0
    m = np.clip(b.min(-1), -big, big).astype(np.float16).astype(np.float64)
    d = np.minimum(np.maximum(b.max(-1) - m, 0.0) / 15.0, big).astype(np.float16).astype(np.float64)
    c = np.where(d[..., None] > 0, np.clip(np.rint((b - m[..., None]) / np.where(d > 0, d, 1.0)[..., None]), 0, 15), 0.0)
    return c.reshape(x.shape), np.where(bad, 0.0, d), np.where(bad, np.nan, m)


def values(c, d, m):
    """What the codes stand for, in 64 bits (exact)."""
    b = c.reshape(*c.shape[:-1], -1, 32)
    return (m[..., None] + d[..., None] * b).reshape(c.shape)


def held(x):
    return values(*quantize(x))


def size(c, d, m):
    """|m| + 15 d of every value's block: what a value's two parts may add up to."""
    return np.repeat(np.abs(m) + 15 * d, 32, -1)


def attention(q, k, v, past, scale):
    """q [n, heads, dim] rotated, k, v [past + n, kv heads, dim] -> out [n, heads, dim], weights [n, heads, past + n]."""
    n, heads, dim = q.shape
    g = heads // k.shape[1]
    out, w = np.zeros(q.shape), np.zeros((n, heads, past + n))
    for t in range(n):
        see = past + t + 1
        for h in range(heads):
            s = k[:see, h // g] @ q[t, h] * scale
            p = np.exp(s - s.max())
            p /= p.sum()
            w[t, h, :see] = p
            out[t, h] = p @ v[:see, h // g]
    return out, w


def tolerance(q_raw, partner, kc, vc, w, past, scale):
    """How far a result in f32 may be from `attention`, [n, heads, dim].

    A score is a sum of q' * (m + d c) with q' in two half-precision parts (together 22 bits, half a step 2^-23) after a rotation in
    f32 (three roundings of 2^-24 of |q| + |partner|) and the scale (two of 2^-24); products of 32 dims are exact and added up in two
    steps that lose at most 2^-22 of the sum of magnitudes each, blocks and parts with a few roundings of 2^-24: together below 2^-20 of
    sum (|q| + |partner|) (|m| + 15 d) scale, the bound e of a score's error. The exponential of it is off by e, the ratio by 2 e.
    Weighted sums lose 2^-22 a step of 16 keys, and of the weights' own parts, joins and the division less than 64 such units."""
    n, heads, dim = q_raw.shape
    g = heads // kc[0].shape[1]
    big_k, big_v = size(*kc), size(*vc)
    tol = np.zeros(q_raw.shape)
    for t in range(n):
        see = past + t + 1
        for h in range(heads):
            e = 2.0 ** -20 * scale * np.nanmax(big_k[:see, h // g] @ (np.abs(q_raw[t, h]) + np.abs(partner[t, h])))
            tol[t, h] = (2 * e + (see / 16 + 64) * 2.0 ** -22) * (w[t, h, :see] @ big_v[:see, h // g])
    return tol


def partners(q, rot, neox):
    """The entry each one is rotated with (0 where none is)."""
    out = np.zeros_like(q)
    if rot:
        a, b = (slice(0, rot // 2), slice(rot // 2, rot)) if neox else (slice(0, rot, 2), slice(1, rot, 2))
        out[..., a], out[..., b] = q[..., b], q[..., a]
    return out
