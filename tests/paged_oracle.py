"""Plain 64-bit forms of the paged KV cache's operators, for the tests: the page
bookkeeping request by request on host lists, decode attention per request and
head in numpy, and how far f32 sums may be from the latter."""
import numpy as np

INT32_MAX = 2**31 - 1


def pages_of(n, ps):
    return -(-n // ps)


def kv_pages(table, old, new, ps, ring, ends, tokens):
    """the step on lists; returns (table, ring, lens, ends, starts, slots, pos)"""
    table = [list(r) for r in table]
    ring = list(ring)
    src = list(ring)
    N, W = len(ring), len(table[0]) if table else 0
    head, tail = ends
    avail = min(max(tail - head, 0), N)
    lens, starts, slots, pos = [], [0], [-1] * tokens, [-1] * tokens
    total = asked = taken = given = 0
    for i, (o, n) in enumerate(zip(old, new)):
        o, n = min(max(o, 0), W * ps), max(n, 0)
        add = max(0, n - o)
        fits = n <= o or (n <= W * ps and total + add <= tokens)
        grow = max(0, pages_of(n, ps) - pages_of(o, ps)) if fits else 0
        ok = fits and (grow == 0 or asked + grow <= avail)
        if ok:
            for k in range(grow):
                table[i][pages_of(o, ps) + k] = src[(head + asked + k) % N]
            taken += grow
            for p in range(o, n):
                page = table[i][p // ps]
                pos[total + p - o] = p
                slots[total + p - o] = page * ps + p % ps if 0 <= page < N else -1
        for k in range(pages_of(n, ps), pages_of(o, ps)):
            ring[(tail + given) % N] = table[i][k]
            given += 1
        lens.append(n if ok else o)
        total += add
        asked += grow
        starts.append(min(total, tokens))
    return table, ring, lens, [head + taken, tail + given], starts, slots, pos


def attn_decode(q, K, V, table, lens, ps, window, scaling):
    """q [R, Hq, D], K and V [pages, ps, Hk, D], all f64 -> (out f64, bound): bound[r, h, d] is how far an
    output may be off. Errors counted, relative to sum_j p_j |v_j|, with u = 2^-24: a score's dot product of D
    f32 products, (D + 1) u sum |q k| scaling at the largest, its scaling and the subtraction of the maximum
    4 u |s|, each entering a weight and, at most as much, the weights' sum (twice), exponentials 4 u, weights
    2^-16, sums of n terms in tiles (a term meets at most 64 additions in its tile and split and 1 a tile or
    split joined: n / 32 + 128) u."""
    R, hq, D = q.shape
    N, _, hk, _ = K.shape
    W = table.shape[1]
    s32 = float(np.float32(scaling))
    out, bound = np.zeros(q.shape), np.zeros(q.shape)
    u = 2.0**-24
    for r in range(R):
        n = min(max(int(lens[r]), 0), W * ps)
        j = np.arange(max(0, n - window) if window > 0 else 0, n)
        page = table[r, j // ps].astype(np.int64)
        live = (page >= 0) & (page < N)
        j, page = j[live], page[live]
        if not len(j):
            continue
        for h in range(hq):
            k, v = (x[page, j % ps, h // (hq // hk)] for x in (K, V))
            s = (k @ q[r, h]) * s32
            p = np.exp(s - s.max())
            p /= p.sum()
            out[r, h] = p @ v
            e = (D + 1) * u * float((np.abs(k) @ np.abs(q[r, h])).max()) * s32 + 8 * u * float(np.abs(s).max())
            bound[r, h] = (2 * e + 8 * u + 2.0**-16 + (len(j) / 32 + 128) * u) * (p @ np.abs(v))
    return out, bound
