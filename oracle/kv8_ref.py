"""The 8-bit paged key/value cache in float64, entry by entry: what it holds, what attention over it gives, what stays after an eviction.

`codes` uint8 [pages, 2, kv_heads, 16 * dim], `scales` [pages, 2, kv_heads]; keys lie [dim / 64][16][64] in a block, values [dim / 64][4][64][4]."""
import numpy as np

PAGE, TOP, LEAST = 16, {"e4m3": 448.0, "int8": 127.0}, -100
LARGEST = {"e4m3": 240.0 * 2.0 ** 120, "int8": 127.0 * 2.0 ** 121}      # code * 2^e within fp32: the next one up is 2^128


def _e4m3_numbers():
    b = np.arange(256)
    x, m = b >> 3 & 15, b & 7
    v = np.where(x == 0, m * 2.0 ** -9, (8 + m) * 2.0 ** (x - 10.0))
    v = np.where(b & 127 == 127, np.nan, v)
    return np.where(b & 128, -v, v)


E4M3 = _e4m3_numbers()


def number(codes, fmt):
    return E4M3[codes] if fmt == "e4m3" else codes.view(np.int8).astype(np.float64)


def code(y, fmt):
    """nearest code, ties to even; beyond the top: the top; NaN: 0"""
    y = np.clip(np.nan_to_num(np.asarray(y, np.float64), nan=0.0, posinf=1e300, neginf=-1e300), -TOP[fmt], TOP[fmt])
    if fmt == "int8":
        return np.rint(y).astype(np.int8).view(np.uint8)
    with np.errstate(divide="ignore"):
        step = 2.0 ** (np.maximum(np.floor(np.log2(np.abs(y))), -6) - 3)
    v = np.rint(y / step) * step
    up = E4M3[:127]
    out = np.searchsorted(up, np.abs(v)).astype(np.uint8)
    assert (up[out] == np.abs(v)).all()
    return np.where(np.signbit(y), out | 128, out).astype(np.uint8)


def exponent(amax, fmt):
    e = LEAST
    while TOP[fmt] * 2.0 ** e < amax:
        e += 1
    return e


def offsets(dim, side, t):
    d = np.arange(dim)
    return d // 64 * 1024 + (t * 64 + d % 64 if side == 0 else t // 4 * 256 + d % 64 * 4 + t % 4)


def page_of(tables, e, block, pages):
    indptr, ids = tables
    n, at = indptr[e + 1] - indptr[e], indptr[e] + block
    if not (0 <= block < n and 0 <= at < len(ids) and 0 <= ids[at] < pages):
        return -1
    return int(ids[at])


def token(codes, scales, fmt, dim, tables, e, slot, side):
    """[kv_heads, dim] values, zeros where the slot has no page"""
    p = page_of(tables, e, slot // PAGE, len(codes))
    if p < 0:
        return np.zeros((codes.shape[2], dim)), False
    return number(codes[p, side][:, offsets(dim, side, slot % PAGE)], fmt) * scales[p, side][:, None].astype(np.float64), True


def append(k, v, codes, scales, fmt, row0, starts, tables):
    """in place"""
    dim = k.shape[2]
    for e in range(len(starts)):
        n, start = row0[e + 1] - row0[e], starts[e]
        for block in range(start // PAGE, (start + n + PAGE - 1) // PAGE if n else 0):
            p = page_of(tables, e, block, len(codes))
            if p < 0:
                continue
            for side, x in enumerate((k, v)):
                for h in range(k.shape[1]):
                    low = block * PAGE
                    old = max(start - low, 0)
                    rows = {t: x[row0[e] + low + t - start, h].astype(np.float64) for t in range(old, PAGE) if start <= low + t < start + n}
                    vals = np.abs(np.concatenate(list(rows.values())))
                    ex = exponent(min(np.max(vals, where=np.isfinite(vals), initial=0.0), LARGEST[fmt]), fmt)
                    was = scales[p, side, h]
                    if old:
                        ex = max(ex, int(np.log2(was)))
                    for t in range(PAGE):
                        at = offsets(dim, side, t)
                        y = number(codes[p, side, h, at], fmt) * (float(was) * 2.0 ** -ex) if t < old else np.clip(rows[t], -LARGEST[fmt], LARGEST[fmt]) * 2.0 ** -ex if t in rows else np.zeros(dim)
                        codes[p, side, h, at] = code(y, fmt)
                    scales[p, side, h] = 2.0 ** ex


def read(codes, scales, fmt, dim, row0, starts, tables):
    out = []
    for side in (0, 1):
        out.append(np.array([token(codes, scales, fmt, dim, tables, e, starts[e] + i, side)[0] for e in range(len(starts)) for i in range(row0[e + 1] - row0[e])]))
    return out


def attention(q, codes, scales, fmt, row0, starts, tables, scale):
    """-> out, weights [entry][kv_heads, slots], and beside every output and weight what its error bound needs: sum p |v| and the largest sum |q k| scale"""
    H, dim = q.shape[1:]
    kv = codes.shape[2]
    out, spread, reach, mass = np.zeros(q.shape), np.zeros(q.shape), np.zeros(q.shape[:2]), []
    for e in range(len(starts)):
        n = row0[e + 1] - row0[e]
        length = starts[e] + n
        got = [[token(codes, scales, fmt, dim, tables, e, s, side) for s in range(length if n else 0)] for side in (0, 1)]
        weight = np.zeros((kv, length if n else 0))
        for i in range(n):
            far = starts[e] + i + 1
            seen = np.array([g[1] for g in got[0][:far]])
            for h in range(H):
                if not seen.any():
                    continue
                K, V = (np.array([g[0][h // (H // kv)] for g in got[side][:far]]) for side in (0, 1))
                x = q[row0[e] + i, h].astype(np.float64)
                z = np.where(seen, K @ x * scale, -np.inf)
                p = np.exp(z - z.max())
                p /= p.sum()
                out[row0[e] + i, h], spread[row0[e] + i, h] = p @ V, p @ np.abs(V)
                reach[row0[e] + i, h] = np.max(np.abs(K) @ np.abs(x)) * abs(scale)
                weight[h // (H // kv), :far] += p
        mass.append(weight)
    return out, mass, spread, reach


def evict(codes, scales, fmt, dim, mass, lens, tables, dst, budget, first, last):
    """in place (codes, scales, mass) -> kept"""
    kv = codes.shape[2]
    kept = np.full((len(lens), kv, budget), -1, np.int32)
    was_codes, was_scales, was_mass = codes.copy(), scales.copy(), mass.copy()
    for e, n in enumerate(lens):
        n = max(0, min(n, PAGE * min(tables[0][e + 1] - tables[0][e], len(tables[1]))))      # no more tokens than its table has places
        for h in range(kv):
            stay = list(range(n))
            if n > budget:
                def key(s):
                    p = page_of(tables, e, s // PAGE, len(codes))
                    m = np.nan if p < 0 else was_mass[p, h, s % PAGE]
                    return (1 if np.isnan(m) else 0, 0.0 if np.isnan(m) else -float(m), s)
                between = sorted(range(first, n - last), key=key)[:budget - first - last]
                stay = sorted(list(range(first)) + between + list(range(n - last, n)))
            kept[e, h, :len(stay)] = stay
            for b in range((len(stay) + PAGE - 1) // PAGE):
                to = page_of(dst, e, b, len(codes))
                if to < 0:
                    continue
                src = [(page_of(tables, e, s // PAGE, len(codes)), s % PAGE) for s in stay[b * PAGE:(b + 1) * PAGE]]
                for side in (0, 1):
                    ex = max([LEAST] + [int(np.log2(was_scales[p, side, h])) for p, _ in src if p >= 0])
                    for t in range(PAGE):
                        y = np.zeros(dim)
                        if t < len(src) and src[t][0] >= 0:
                            p, ts = src[t]
                            y = number(was_codes[p, side, h, offsets(dim, side, ts)], fmt) * (float(was_scales[p, side, h]) * 2.0 ** -ex)
                        codes[to, side, h, offsets(dim, side, t)] = code(y, fmt)
                    scales[to, side, h] = 2.0 ** ex
                for t in range(PAGE):
                    mass[to, h, t] = was_mass[src[t][0], h, src[t][1]] if t < len(src) and src[t][0] >= 0 else 0.0
    return kept
