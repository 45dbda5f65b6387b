"""The paged operators and norm_rotary from their formulas, in numpy float64, one
row at a time; and bounds of what rounding does to them."""

import numpy as np


def length_of(lengths, b, width, size):
    return int(min(max(int(lengths[b]), 0), width * size))


def slots(table, n, size, num_pages):
    """(slot, named) of positions 0..n-1 of one page table."""
    ids = np.asarray([int(table[j // size]) for j in range(n)], dtype=np.int64)
    named = (ids >= 0) & (ids < num_pages)
    return np.where(named, ids, 0) * size + np.arange(n) % size, named


def attention(table, lengths, size, num_pages, queries, q, k, v, scale):
    """q [rows, heads, group, D]; k, v [slots, heads, D]; table [B, P], or
    [B, T, P] with rows of (b, t, table head) and caches [slots, T, heads, D]."""
    table = np.asarray(table)
    per_head = table.ndim == 3
    tables = table if per_head else table[:, None]
    B, T, P = tables.shape
    heads, group = q.shape[1:3]
    out = np.zeros(q.shape)
    for b in range(B):
        for t in range(queries):
            n = max(length_of(lengths, b, P, size) - (queries - 1 - t), 0)
            for th in range(T):
                row = (b * queries + t) * T + th
                at, named = slots(tables[b, th], n, size, num_pages)
                at = at[named]
                if at.size == 0:
                    continue
                for h in range(heads):
                    kk, vv = (x[at, th, h] if per_head else x[at, h] for x in (k, v))
                    s = scale * (q[row, h] @ kk.T)
                    w = np.exp(s - s.max(-1, keepdims=True))
                    out[row, h] = (w / w.sum(-1, keepdims=True)) @ vv
    return out


def select(table, lengths, size, num_pages, queries, q, sums, count):
    """(page table [rows, heads, count], lengths [rows])."""
    rows, heads = q.shape[:2]
    out = np.full((rows, heads, count), -1, dtype=np.int32)
    kept_lengths = np.zeros(rows, dtype=np.int32)
    for row in range(rows):
        b, t = divmod(row, queries)
        n = max(length_of(lengths, b, table.shape[1], size) - (queries - 1 - t), 0)
        pages = -(-n // size)
        if pages == 0:
            continue
        kept = min(pages, count)
        kept_lengths[row] = (kept - 1) * size + n - (pages - 1) * size
        for h in range(heads):
            summed = q[row, h].sum(0)
            score = []
            for p in range(pages - 1):
                i = int(table[b, p])
                x = float(summed @ sums[i, h]) if 0 <= i < num_pages else -np.inf
                score.append(-np.inf if np.isnan(x) else x)
            best = sorted(range(pages - 1), key=lambda p: (-score[p], p))[:kept - 1]
            out[row, h, :kept] = [table[b, p] for p in sorted(best) + [pages - 1]]
    return out, kept_lengths


def append(table, lengths, size, num_pages, queries, kc, k, vc, v, sums=None):
    """The caches (copies) and page sums after the append."""
    kc, vc = kc.copy(), vc.copy()
    sums = None if sums is None else sums.astype(np.float64)
    for b in range(table.shape[0]):
        n = length_of(lengths, b, table.shape[1], size)
        touched = set()
        for t in range(queries):
            pos = n - queries + t
            if pos < 0 or not 0 <= table[b, pos // size] < num_pages:
                continue
            slot = int(table[b, pos // size]) * size + pos % size
            kc[slot], vc[slot] = k[b * queries + t], v[b * queries + t]
            touched.add(pos // size)
        if sums is not None:
            for p in touched:
                first = int(table[b, p]) * size
                held = min(n - p * size, size)
                sums[table[b, p]] = kc[first:first + held].astype(np.float64).sum(0)
    return kc, vc, sums


def rotate(u, angle, interleaved, sign=1.0):
    half = angle.shape[-1]
    y = u.copy()
    first = slice(0, 2 * half, 2) if interleaved else slice(0, half)
    second = slice(1, 2 * half, 2) if interleaved else slice(half, 2 * half)
    c, s = np.cos(angle)[:, None], sign * np.sin(angle)[:, None]
    y[..., first] = u[..., first] * c - u[..., second] * s
    y[..., second] = u[..., second] * c + u[..., first] * s
    return y


def angles(positions, freqs, sections):
    axis = np.repeat(np.arange(len(sections)), sections)
    return positions.astype(np.float64)[:, axis] * freqs.astype(np.float64)


def norm_rotary(x, w, angle, eps, norm, interleaved):
    n = x / np.sqrt((x ** 2).mean(-1, keepdims=True) + eps) if norm else x
    return rotate(n * w if norm and w is not None else n, angle, interleaved)


def norm_rotary_grad(x, w, angle, eps, norm, interleaved, dy):
    """(dx, dw)"""
    g = rotate(dy, angle, interleaved, -1.0)
    if not norm:
        return g, None
    r = 1 / np.sqrt((x ** 2).mean(-1, keepdims=True) + eps)
    n = x * r
    h = g if w is None else g * w
    return r * (h - n * (h * n).mean(-1, keepdims=True)), (g * n).sum((0, 1))


def attention_bound(table, lengths, size, num_pages, queries, q, k, v, scale, dtype, tiles):
    """What rounding may do to each value of `attention` (shapes as there, one
    table a sequence), by the row's own weights p:

        step |out| + sum_j p_j |v_j| (parts + adds) + 2 sum_j p_j ds_j (|v_j| + |out|)

    step: half a step of the output's type; parts: a weight as two 16-bit values
    (`tiles`: the matrix kernels; fp16's may be off by 2^-39 of the largest as
    well), or in fp32; adds: two fp32 roundings for each addition one after the other
    (a key at a time on a quarter of the row at least, 32 keys at a time in a
    tile), and 64 for waves, pieces and exponentials; ds_j: the fp32 score's D
    products and its scaling."""
    f32 = 2.0 ** -24
    step = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}[dtype]
    parts = 2 * step ** 2 if tiles else f32
    table = np.asarray(table)
    heads, group, D = q.shape[1:]
    lim = np.zeros(q.shape)
    for b in range(table.shape[0]):
        for t in range(queries):
            row = b * queries + t
            n = max(length_of(lengths, b, table.shape[1], size) - (queries - 1 - t), 0)
            at, named = slots(table[b], n, size, num_pages)
            at = at[named]
            if at.size == 0:
                continue
            adds = 2 * f32 * (n / (32 if tiles else 4) + 64)
            for h in range(heads):
                kk, vv = k[at, h], np.abs(v[at, h])
                s = scale * (q[row, h] @ kk.T)
                p = np.exp(s - s.max(-1, keepdims=True))
                p /= p.sum(-1, keepdims=True)
                out = np.abs(p @ v[at, h])
                ds = f32 * ((D + 8) * abs(scale) * (np.abs(q[row, h]) @ np.abs(kk).T) +
                            4 * np.abs(s))
                lim[row, h] = step * out + (parts + adds) * (p @ vv) + \
                    2 * ((p * ds) @ vv + (p * ds).sum(-1, keepdims=True) * out)
                if tiles and dtype == "f16":
                    lim[row, h] += 2.0 ** -39 * vv.sum(0)
    # (Outputs below the type's normal numbers round in absolute steps.)
    tiny = {"f32": 2.0 ** -149, "bf16": 2.0 ** -133, "f16": 2.0 ** -24}[dtype]
    return lim + tiny
