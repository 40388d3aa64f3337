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


def rms_tolerance(q, q_raw, partner, kc, vc, w, past, scale):
    """Six standard deviations of what the roundings of an attention in f32 with factors of 22 bits make of `attention`, [n, heads, dim], where
    `tolerance` adds up their worst cases. q is rotated, q_raw is not. To first order in errors that know nothing of one another, with s the scores, o the
    output and C[i, i'] = sum_j w_j (v_ji - o_i) k_ji':

    * an entry of a query is off by up to 6 * 2^-24 of |q| + |partner| (rotation 3, scale 1, pair of half-precision numbers 2), for all keys alike: by C;
    * a key's score besides by 2^-21 of the root of the sum of squares of (|q| + |partner|) (|m| + 15 d) scale (a term's two products, their
      alignment in sums of 16 and 32), by 2^-22 of its and the largest score's magnitude (the reference, the argument of the exponential), its exponential by 2^-22;
    * all scores alike by 2^-22 of themselves (the scale and log2 e as f32 numbers);
    * a weighted value by 2^-20 of |m| + 15 d (pairs 2^-22, alignment in up to 16 steps of a sum before it joins an f32 one);
    and the output by 2^-22 of itself (joins, division)."""
    n, heads, dim = q.shape
    g = heads // kc[0].shape[1]
    (k, v), (big_k, big_v) = (values(*kc), values(*vc)), (size(*kc), size(*vc))
    tol = np.zeros(q.shape)
    for t in range(n):
        see = past + t + 1
        for h in range(heads):
            p, kh, vh, aq = w[t, h, :see], k[:see, h // g], v[:see, h // g], np.abs(q_raw[t, h]) + np.abs(partner[t, h])
            o, s = p @ vh, scale * (kh @ q[t, h])
            far = vh - o                                       # [see, dim]
            each = 2.0 ** -21 * scale * np.sqrt((big_k[:see, h // g] ** 2) @ (aq ** 2)) + 2.0 ** -22 * (np.abs(s) + np.abs(s).max() + 1)
            var = (6 * 2.0 ** -24 * scale) ** 2 * ((p[:, None] * far).T @ kh) ** 2 @ (aq ** 2) + (p * each) ** 2 @ far ** 2
            var += (2.0 ** -22 * ((p * s) @ far)) ** 2 + 2.0 ** -40 * (p ** 2 @ big_v[:see, h // g] ** 2)
            tol[t, h] = 6 * np.sqrt(var) + 2.0 ** -22 * np.abs(o)
    return tol


def half_pair(x, parts=2):
    """64-bit numbers as one half-precision number or the sum of two (value and remainder)."""
    hi = x.astype(np.float16).astype(np.float64)
    return hi if parts == 1 else hi + (x - hi).astype(np.float16).astype(np.float64)


def attention_in_halves(q, kc, vc, past, scale, q_parts=2, w_parts=2, by_block=True):
    """`attention` with queries and weight * step as half-precision operands, all else in 64 bits: queries scaled to below 2^10, steps to below 1 by a power of two for
    each block of 32 dims (or one for all of them, as steps in half precision then), weights from 2^7 down. One part of an operand shows what its remainder is worth."""
    n, heads, dim = q.shape
    g = heads // kc[0].shape[1]
    k, (c, d, m) = values(*kc), vc
    out = np.zeros(q.shape)
    down = lambda x: 2.0 ** np.floor(np.log2(np.where(x > 0, x, 1.0)))
    for t in range(n):
        see = past + t + 1
        for h in range(heads):
            lift = down(np.abs(q[t, h]).max()) / 2.0 ** 9
            s = k[:see, h // g] @ (half_pair(q[t, h] / lift, q_parts) * lift) * scale
            p = np.exp(s - s.max()) * 2.0 ** 7
            dh, mh = d[:see, h // g], m[:see, h // g]
            top = 2 * (down(dh.max(0)) if by_block else down(np.full(dh.shape[1], dh.max())))
            step = dh / top if by_block else (dh / top).astype(np.float16).astype(np.float64)
            w = half_pair(p[:, None] * step, w_parts) * top
            o = ((np.repeat(w, 32, 1) * (c[:see, h // g] - 8)).reshape(see, -1).sum(0) + np.repeat(p @ (mh + 8 * dh), 32)) / p.sum()
            out[t, h] = o
    return out
