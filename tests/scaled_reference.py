"""Caches in 8 bits, and attention over a window, from their formulas in numpy
float64; and bounds of what rounding does to them."""

import numpy as np

from paged_reference import length_of, slots

LARGEST = {"e4m3": 448.0, "int8": 127.0}


def scale_of(amax, code):
    """The smallest power of two s >= 2^-126 with amax <= M s."""
    if not np.isfinite(amax):
        return np.nan
    s = 2.0 ** -126
    while amax > LARGEST[code] * s:
        s *= 2.0
    return s


def rounded(x, code):
    """Values to the nearest code, ties to even: steps of 1, or of 2^(e - 3)
    between 2^e and 2^(e + 1), and of 2^-9 below 2^-6."""
    if code == "int8":
        return np.rint(x)
    e = np.floor(np.log2(np.maximum(np.abs(x), 2.0 ** -6)))
    step = 2.0 ** (e - 3)
    return np.rint(x / step) * step


def append(table, lengths, size, num_pages, queries, codes, scales, new, code, block):
    """(codes as numbers, scales) after an append of `new` [rows, heads, D]."""
    codes, scales = codes.copy(), scales.copy()
    for b in range(table.shape[0]):
        n = length_of(lengths, b, table.shape[1], size)
        fresh = max(n - queries, 0)
        for first in range(fresh // block * block, n, block):
            page = int(table[b, first // size])
            if not 0 <= page < num_pages:
                continue
            slot = page * size + first % size
            low, high = max(first, fresh) - first, min(n - first, block)
            x = new[b * queries + first + low - (n - queries):
                    b * queries + first + high - (n - queries)]
            for h in range(new.shape[1]):
                s = scale_of(np.abs(x[:, h]).max(), code)
                held = scales[slot // block, h]
                if low:
                    s = np.nan if np.isnan(s) or np.isnan(held) else max(s, held)
                    if not np.isnan(s):
                        codes[slot:slot + low, h] = rounded(codes[slot:slot + low, h] * (held / s),
                                                            code)
                scales[slot // block, h] = s
                codes[slot + low:slot + high, h] = 0 if np.isnan(s) else rounded(x[:, h] / s, code)
    return codes, scales


def values(codes, scales, block):
    return codes * np.repeat(scales, block, 0)[:, :, None]


def read(table, lengths, size, num_pages, queries, rows):
    """The newest tokens' rows [sequences * queries, heads, D] of `rows` [slots, ...]."""
    out = np.zeros((table.shape[0] * queries, *rows.shape[1:]))
    for b in range(table.shape[0]):
        n = length_of(lengths, b, table.shape[1], size)
        for t in range(queries):
            pos = n - queries + t
            if pos >= 0 and 0 <= table[b, pos // size] < num_pages:
                out[b * queries + t] = rows[int(table[b, pos // size]) * size + pos % size]
    return out


def page_sums(table, lengths, size, num_pages, queries, rows, sums):
    sums = sums.astype(np.float64)
    for b in range(table.shape[0]):
        n = length_of(lengths, b, table.shape[1], size)
        for p in range(max(n - queries, 0) // size, -(-n // size)):
            if 0 <= table[b, p] < num_pages:
                first = int(table[b, p]) * size
                sums[table[b, p]] = rows[first:first + min(n - p * size, size)].sum(0)
    return sums


def seen(n, window, sinks):
    """Positions that the newest of n tokens sees."""
    at = np.arange(max(n, 0))
    return at if window is None else at[(at >= n - window) | (at < sinks)]


def paged_attention(table, lengths, size, num_pages, queries, q, k, v, scale, window=None, sinks=0,
                    tiles=None, step=0.0, part=0.0):
    """(out, bound): q [rows, heads, group, D], k and v [slots, heads, D].

    bound, by the row's own weights p, of keys that are exact: `step` (half a step of
    the output's type) of the output; `part` of sum p |v| for what each weight is
    rounded to (two 16-bit parts of the type the values are multiplied in, or fp32),
    and 2^-24 for each of the additions, key by key or 32 keys at a time (`tiles`), with
    64 for waves, pieces, exponentials and scales; and the fp32 scores' D products."""
    f32 = 2.0 ** -24
    heads, group, D = q.shape[1:]
    out, lim = np.zeros(q.shape), np.zeros(q.shape)
    for b in range(table.shape[0]):
        for t in range(queries):
            row = b * queries + t
            n = length_of(lengths, b, table.shape[1], size) - (queries - 1 - t)
            pos = seen(n, window, sinks)
            if pos.size == 0:
                continue
            at, named = slots(table[b], n, size, num_pages)
            at = at[pos][named[pos]]
            if at.size == 0:
                continue
            adds = 2 * f32 * (at.size / (32 if tiles else 4) + 64)
            for h in range(heads):
                kk, vv = k[at, h], v[at, h]
                s = scale * (q[row, h] @ kk.T)
                with np.errstate(invalid="ignore"):
                    p = np.exp(s - s.max(-1, keepdims=True))
                    p /= p.sum(-1, keepdims=True)
                    out[row, h] = p @ vv
                ds = f32 * ((D + 10) * abs(scale) * (np.abs(q[row, h]) @ np.abs(kk).T) +
                            4 * np.abs(s))
                near = np.abs(out[row, h])
                lim[row, h] = step * near + (part + adds) * (p @ np.abs(vv)) + \
                    2 * ((p * ds) @ np.abs(vv) + (p * ds).sum(-1, keepdims=True) * near)
    return out, lim


def window_attention(lengths, q, k, v, scale, window, sinks, dout=None, half=0.0):
    """Packed sequences: q, dout [n, heads, group, D], k and v [n, heads, D].
    ((out, dq, dk, dv), their bounds), out alone without dout.

    The bounds: half a step (`half`) of each result; P and dS rounded to the inputs' type
    (half a step each), delta from the rounded output; fp32 sums of up to n + D products,
    and scores that are off by ds relative to p.  The denominator is a sum of rounded
    weights, sum_j w_j (1 + d_j) with |d_j| <= half: off by a factor of 1 + e, |e| <=
    half, which the backward's P = w / sum carries in full (beside its own rounding),
    and dS = P (dP - delta) with it."""
    f32 = 2.0 ** -24
    n, heads, group, D = q.shape
    shapes = (q.shape, q.shape, k.shape, v.shape)
    res = [np.zeros(s) for s in shapes]
    lim = [np.zeros(s) for s in shapes]
    start = 0
    for length in lengths:
        rows = slice(start, start + length)
        i, j = np.arange(length)[:, None], np.arange(length)
        mask = (j <= i) & ((i - j < window) | (j < sinks))
        for h in range(heads):
            kk, vv = k[rows, h], v[rows, h]
            for g in range(group):
                qq = q[rows, h, g]
                s = np.where(mask, scale * (qq @ kk.T), -np.inf)
                if length == 0:
                    continue
                p = np.exp(s - s.max(-1, keepdims=True))
                p /= p.sum(-1, keepdims=True)
                out = p @ vv
                adds = 2 * f32 * (length + 64)
                # A weight's relative error: its score's absolute one (of the row's own
                # and of its logarithmic sum), and its rounding.
                ds_ = f32 * ((D + 10) * abs(scale) * (np.abs(qq) @ np.abs(kk).T) +
                             8 * np.abs(np.where(mask, s, 0)) + 16)
                rel = 2 * (ds_ + np.where(mask, ds_, 0).max(-1, keepdims=True)) + adds
                res[0][rows, h, g] = out
                out_lim = half * np.abs(out) + (p * (rel + half)) @ np.abs(vv) + \
                    (p * half).sum(-1, keepdims=True) * np.abs(out)
                lim[0][rows, h, g] = out_lim
                if dout is None:
                    continue
                d = dout[rows, h, g]
                dp = d @ vv.T
                delta = (d * out).sum(-1, keepdims=True)
                ds = p * (dp - delta)
                res[1][rows, h, g] = scale * ds @ kk
                res[2][rows, h] += scale * ds.T @ qq
                res[3][rows, h] += p.T @ d
                size = np.abs(d) @ np.abs(vv).T + (np.abs(d) * np.abs(out)).sum(-1, keepdims=True)
                e_p = p * (rel + 2 * half)
                e_ds = half * np.abs(ds) + p * ((rel + half) * np.abs(dp - delta) +
                                                (D + 8) * f32 * size +
                                                (np.abs(d) * out_lim).sum(-1, keepdims=True))
                more = adds * group * p
                lim[1][rows, h, g] = half * np.abs(res[1][rows, h, g]) + \
                    abs(scale) * (e_ds + adds * np.abs(ds)) @ np.abs(kk)
                lim[2][rows, h] += abs(scale) * (e_ds + adds * group * np.abs(ds)).T @ np.abs(qq)
                lim[3][rows, h] += (e_p + more).T @ np.abs(d)
        start += length
    if dout is None:
        return res[0], lim[0]
    for x in (2, 3):
        lim[x] += half * np.abs(res[x])
    return res, lim
