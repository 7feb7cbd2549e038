"""Definitions in whole numbers of the operators around attention and the pick (include/sslm_b200.h)."""
import math

import numpy as np

PAGE = 16
LOWEST = -(1 << 31)
EXP2 = (2147483648, 1488326151, 514119776, 114090822, 14555373)


# ------------------------------------------------------------------------------- the q/k/v site
def rounded(num, den):
    """num / den to the nearest, halves away from zero (den > 0)."""
    return (2 * abs(num) + den) // (2 * den) * (1 if num >= 0 else -1)


def held(x):
    return max(-127, min(127, x))


def canonical(m, e):
    while m < 1 << 30:
        m, e = 2 * m, e - 1
    return m, e


def combine(a, b):
    return canonical((a[0] * b[0] + (1 << 30)) >> 31, a[1] + b[1] + 31)


def scale_of(x):
    f, e = math.frexp(x)
    m = int(round(f * (1 << 31)))
    return (m, e - 31) if m < 1 << 31 else (m >> 1, e - 30)


def reciprocal(m):
    return ((1 << 62) + m // 2) // m


def normed(x, gain, shift):
    top = max(abs(v) for v in x)
    if top == 0:
        return [0] * len(x)
    up = 24 - top.bit_length()
    y = [v << up if up >= 0 else rounded(v, 1 << -up) for v in x]
    root = math.isqrt(64 * sum(v * v for v in y) // len(y))
    return [rounded(rounded(v * ((1 << 54) // root), 1 << 36) * int(g), 1 << shift) for v, g in zip(y, gain)]


def landed(x, scale, rec):
    cut = 62 - (scale[1] - rec[1])
    num = scale[0] * rec[2]
    return [rounded(v * num, 1 << cut) if cut >= 0 else v * num << -cut for v in x]


def turned(x, cos, sin, halves):
    x, n = list(x), len(cos)
    for i in range(n):
        a, b = (i, i + n) if halves else (2 * i, 2 * i + 1)
        c, s = int(cos[i]), int(sin[i])
        x[a], x[b] = held(rounded(x[a] * c - x[b] * s, 1 << 30)), held(rounded(x[a] * s + x[b] * c, 1 << 30))
    return x


def softmax_constants(out, khead):
    m, e = combine(out, khead)
    r = reciprocal(m)
    if 92 + e < 0 or 154 + 2 * e < 0:
        return (0, 0, 0)
    c = 744261117 * r >> (92 + e), 1452772687 * r >> (92 + e), r * r * 1030312935 >> (154 + 2 * e)
    return c if all(v < 1 << 63 for v in c) and c[0] >= 1 and c[1] ** 2 + c[2] <= (1 << 62) >> 15 else (0, 0, 0)


def site_case(seed, shape, rows, positions=64, rotary=None, halves=False, norm="", tables=None, deviation=20000.0, spare=2):
    """Rows at places that differ; every row a table of its own unless `tables` are fewer."""
    H, KVH, hd = shape
    g = np.random.default_rng(seed)
    rotary = hd if rotary is None else rotary
    tables = rows if tables is None else tables
    width = -(-positions // PAGE)
    wide = np.clip(np.rint(g.normal(0, deviation, (rows, (H + 2 * KVH) * hd))), LOWEST, -LOWEST - 1).astype(np.int32)
    table_of = np.arange(rows) % tables
    place = np.zeros(rows, dtype=np.int64)
    for s in range(tables):
        mine = np.flatnonzero(table_of == s)
        place[mine] = g.choice(width * PAGE, len(mine), replace=False)
    angle = np.arange(positions)[:, None] * 1e4 ** (-np.arange(rotary // 2)[None, :] / max(1, rotary // 2))
    in_scales = np.stack([g.integers(1 << 30, 1 << 31, rows), g.integers(-51, -48, rows)], 1)

    def landing():
        recs = []
        for _ in range(KVH):
            m, e = scale_of(2.0 ** -19.5 * max(1.0, deviation) / 32.0 * g.uniform(0.5, 1.5))
            recs.append((m, e, reciprocal(m)))
        return np.array(recs, dtype=np.int64)
    return dict(wide=wide, in_scales=in_scales.astype(np.int64), positions=g.integers(0, positions, rows).astype(np.int32), places=place.astype(np.int32),
                table_of=table_of.astype(np.int32), pages=g.permutation(tables * width + spare)[:tables * width].reshape(tables, width).astype(np.int32),
                kv=g.integers(-127, 128, (KVH, 2, tables * width + spare, PAGE * hd)).astype(np.int8),
                cos=np.rint(np.cos(angle) * (1 << 30)).astype(np.int32).reshape(positions, rotary // 2), sin=np.rint(np.sin(angle) * (1 << 30)).astype(np.int32).reshape(positions, rotary // 2),
                k_landing=landing(), v_landing=landing(), q_site=scale_of(1.0 / 127),
                khead=np.array([scale_of(g.uniform(1, 2) / (1600.0 * math.sqrt(hd)) / (2.0 ** -19.5 * max(1.0, deviation) * 4 / 127)) for _ in range(KVH)], dtype=np.int64),
                q_gain=g.integers(-9000, 9000, hd).astype(np.int16) if "q" in norm else None, k_gain=g.integers(-9000, 9000, hd).astype(np.int16) if "k" in norm else None,
                q_shift=23, k_shift=22, halves=halves, shape=shape)


def site_rows(c, only=None):
    """{row: (q codes, q scale, constants, saturations, K codes, V codes)}"""
    H, KVH, hd = c["shape"]
    out = {}
    for r in range(len(c["wide"])) if only is None else only:
        x = [int(v) for v in c["wide"][r]]
        heads = [x[i * hd:(i + 1) * hd] for i in range(H + 2 * KVH)]
        q, k, v = heads[:H], heads[H:H + KVH], heads[H + KVH:]
        scale, pos = tuple(int(t) for t in c["in_scales"][r]), int(c["positions"][r])
        if c["q_gain"] is not None:
            codes, qs = [normed(t, c["q_gain"], c["q_shift"]) for t in q], c["q_site"]
        else:
            top = max([1] + [abs(t) for row in q for t in row])
            up = 31 - top.bit_length()
            d = top << up if up >= 0 else top >> -up
            codes = [[min(127, (abs(t) * reciprocal(d) * 127 + (1 << (61 - up))) >> (62 - up)) * (1 if t > 0 else -1) for t in row] for row in q]
            qs = combine(combine(scale, c["q_site"]), (d, -up))
        cs, sn = c["cos"][pos], c["sin"][pos]
        K = [normed(t, c["k_gain"], c["k_shift"]) if c["k_gain"] is not None else landed(t, scale, [int(u) for u in c["k_landing"][h]]) for h, t in enumerate(k)]
        V = [landed(t, scale, [int(u) for u in c["v_landing"][h]]) for h, t in enumerate(v)]
        sat = sum(abs(t) > 127 for row in K + V for t in row)
        out[r] = (np.array([turned([held(t) for t in row], cs, sn, c["halves"]) for row in codes]).reshape(H, hd), qs,
                  np.array([softmax_constants(qs, tuple(int(t) for t in c["khead"][h])) for h in range(KVH)]), sat,
                  np.array([turned([held(t) for t in row], cs, sn, c["halves"]) for row in K]), np.array([[held(t) for t in row] for row in V]))
    return out


# ------------------------------------------------------------------------------------ the draw
def weights(d, slope, cut):
    """of distances d (int64, below 2^32) from the largest logit"""
    t = (d * np.int64(slope)) >> np.int64(cut)                # (below 2^63)
    f = (t & 0xFFFFFF).astype(np.uint64) << np.uint64(8)
    p = np.full(len(t), EXP2[4], dtype=np.uint64)
    for c in EXP2[3::-1]:
        p = np.uint64(c) - (f * p >> np.uint64(32))
    return np.where(t < 32 << 24, (p >> np.minimum(t >> 24, 63).astype(np.uint64)).astype(np.int64), 0)


def drawn(x, slope, cut, top_k, top_p, min_p, draw):
    """(token, its weight, sum of the kept, how many) of one row of logits"""
    ids = np.flatnonzero(x != LOWEST)
    if len(ids) == 0:
        return -2, 0, 0, 0
    x = x.astype(np.int64)
    ids = ids[np.lexsort((ids, -x[ids]))]
    d = x[ids[0]] - x[ids]
    w = weights(d, slope, cut)
    if top_k:
        ids, w = ids[:top_k], w[:top_k]
    enough = int(w.sum()) * top_p >> 30
    keep = (np.cumsum(w) - w < enough) & (w >= 2 * min_p) & (w > 0)
    ids, w = ids[keep], w[keep]
    back = np.argsort(ids)
    ids, w = ids[back], w[back]
    total = int(w.sum())
    at = int(np.searchsorted(np.cumsum(w), total * draw >> 31, side="right"))
    return int(ids[at]), int(w[at]), total, len(ids)


# ----------------------------------------------------------------------------------- the pages
def cache_case(seed, sequences, longest, pages=None, planes=3, page_bytes=48, shared=True, grow=0, spare=5):
    """Tables of sequences with prefixes in common, and a pool."""
    g = np.random.default_rng(seed)
    width = max(1, -(-(longest + grow) // PAGE))
    need = sequences * (-(-longest // PAGE) + 1) + spare
    pages = need if pages is None else pages
    lengths = g.integers(0, longest + 1, sequences).astype(np.int32)
    free = iter(g.permutation(pages).tolist())
    tables, holders = np.full((sequences, width), -7, dtype=np.int32), np.zeros(pages, dtype=np.int32)
    for i in range(sequences):
        used = -(-int(lengths[i]) // PAGE)
        n = int(min(lengths[i - 1], lengths[i])) // PAGE // 2 if shared and i % 2 else 0
        tables[i, :n] = tables[i - 1, :n]
        tables[i, n:used] = [next(free) for _ in range(used - n)]
        np.add.at(holders, tables[i, :used], 1)
    return dict(kv=g.integers(-128, 128, (planes, pages, page_bytes)).astype(np.int8), holders=holders, tables=tables, lengths=lengths)


def forked(c, parents, grow, out_tables):
    """What sslm_b200_fork_resident leaves: a dict of arrays, out_tables begun with."""
    n, width = c["tables"].shape
    N = len(c["holders"])
    free = [p for p in range(N) if c["holders"][p] == 0]
    held_by, tables, lengths = c["holders"].astype(np.int64), out_tables.copy(), np.zeros(n, dtype=np.int32)
    status, moves, asked, taken, kv = np.zeros(n, dtype=np.int32), [], 0, 0, c["kv"].copy()
    room = width * PAGE

    def pages_of(i):
        m = int(c["lengths"][i])
        return c["tables"][i, :-(-m // PAGE)].tolist() if 0 <= m <= room else []
    for i in range(n):
        p, more = int(parents[i]), int(grow[i])
        code, keep, fresh = 0, [], 0
        if p < -1 or p >= n:
            code = 101
        elif p >= 0:
            m = int(c["lengths"][p])
            if m < 0 or more < 0 or m + more > room:
                code = 7
            elif p != i and any(not 0 <= q < N for q in pages_of(p)):
                code = 101
            else:
                keep = pages_of(p)[:m // PAGE if p != i else None]
                fresh = -(-(m + more) // PAGE) - len(keep)
                if fresh and asked + fresh > len(free):
                    code = 102
                asked += fresh
        status[i] = code
        if code:
            lengths[i] = c["lengths"][i]
            own = pages_of(i)
            tables[i, :len(own)] = own
            continue
        if p != i:
            for q in pages_of(i):
                if 0 <= q < N:
                    held_by[q] -= 1
        if p < 0:
            continue
        lengths[i] = m + more
        new = free[asked - fresh:asked]
        taken += fresh
        if p != i and m % PAGE:
            moves.append((pages_of(p)[m // PAGE], new[0]))
        for q in keep if p != i else []:
            held_by[q] += 1
        for q in new:
            held_by[q] += 1
        tables[i, :len(keep) + fresh] = keep + new
    for a, b in moves:
        kv[:, b] = c["kv"][:, a]
    return dict(out_holders=held_by.astype(np.int32), out_tables=tables, out_lengths=lengths, status=status, kv=kv, moves=np.array(moves, dtype=np.int32).reshape(-1, 2),
                drawn=np.array(free[:taken], dtype=np.int32))


def compacted(c, out_tables):
    n, width = c["tables"].shape
    N = len(c["holders"])
    used = [p for p in range(N) if c["holders"][p] != 0]
    holes = [p for p in range(len(used)) if c["holders"][p] == 0]
    moves = list(zip([p for p in used if p >= len(used)], holes))
    new = {p: p for p in used if p < len(used)}
    new.update(moves)
    new_of, held_by, kv, tables, status = np.full(N, -1, dtype=np.int32), np.zeros(N, dtype=np.int32), c["kv"].copy(), out_tables.copy(), np.zeros(n, dtype=np.int32)
    for a, b in new.items():
        new_of[a], held_by[b] = b, c["holders"][a]
    for a, b in moves:
        kv[:, b] = c["kv"][:, a]
    for i in range(n):
        m = int(c["lengths"][i])
        if not 0 <= m <= width * PAGE:
            status[i] = 7
            continue
        own = c["tables"][i, :-(-m // PAGE)].tolist()
        if any(not 0 <= p < N or new_of[p] < 0 for p in own):
            status[i] = 101
        else:
            tables[i, :len(own)] = [new_of[p] for p in own]
    return dict(out_holders=held_by, out_tables=tables, new_of=new_of, status=status, kv=kv, moves=np.array(moves, dtype=np.int32).reshape(-1, 2), live=len(used))
