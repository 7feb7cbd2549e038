"""Inputs and 64-bit definitions of the operators on a caller's tensors (include/sslm_b200.h)."""
import numpy as np

PAGE = 16
LOWEST = -(1 << 31)


def attention_case(seed, shape, prefix, suffix, per_group=None, deviation=40.0, consts=None, spare_pages=3, widths=(0, 0)):
    """prefix: positions of each group; suffix: positions of each row; per_group: rows of each group (default: even);
    widths: pages that the tables have room for at least, those behind a length without a page (-1)."""
    heads, kv_heads, hd = shape
    g = np.random.default_rng(seed)
    rows, groups = len(suffix), len(prefix)
    if per_group is None:
        per_group = [rows // groups + (i < rows % groups) for i in range(groups)]
    start = np.concatenate([[0], np.cumsum(per_group)]).astype(np.int32)
    pp = max([1] + [-(-p // PAGE) for p in prefix])
    sp = max([1] + [-(-s // PAGE) for s in suffix])
    pages = groups * pp + rows * sp + spare_pages
    order = g.permutation(pages).astype(np.int32)

    def codes(n):
        return np.clip(np.rint(g.normal(0, deviation, n)), -128, 127).astype(np.int8)
    if consts is None:
        scale = g.uniform(1, 3, (rows, kv_heads)) / (max(1.0, deviation) ** 2 * np.sqrt(hd))
        consts = np.stack([np.floor(np.log(2) / scale), np.floor(1.353 / scale), np.floor(0.9595 / scale ** 2)], -1).astype(np.int64)
    else:
        consts = np.broadcast_to(np.asarray(consts, dtype=np.int64), (rows, kv_heads, 3)).copy()
    fold = np.zeros((heads, 3), dtype=np.int32)
    fold[:, 1] = g.integers(-(1 << 31) + 1, (1 << 31) - 1, heads)
    fold[:, 2] = g.integers(0, 12, heads)
    fold[::3, 0] = 1
    def table(ids, width):
        return np.concatenate([ids, np.full((len(ids), max(0, width - ids.shape[1])), -1, dtype=np.int32)], axis=1)
    return dict(q=codes((rows, heads, hd)), consts=consts, kv=codes((kv_heads, 2, pages, PAGE * hd)), group_start=start,
                prefix_len=np.asarray(prefix, dtype=np.int32), prefix_pages=table(order[:groups * pp].reshape(groups, pp), widths[0]),
                suffix_len=np.asarray(suffix, dtype=np.int32), suffix_pages=table(order[groups * pp:groups * pp + rows * sp].reshape(rows, sp), widths[1]), fold=fold)


def fold64(x, identity, mult, shift):
    if identity:
        return x
    x = np.minimum((x * int(mult) + (1 << 30)) >> 31, (1 << 31) - 1)
    rest = x & ((1 << int(shift)) - 1)
    return (x >> int(shift)) + (rest > ((((1 << int(shift)) - 1) >> 1) + (x < 0)))


def attention_rows(c, only=None):
    """{row: int64 [heads, hd]} of the rows that lie in a group."""
    rows, heads, hd = c["q"].shape
    kv = c["kv"]
    KVH = kv.shape[0]
    G = heads // KVH
    want = {}
    for g in range(len(c["prefix_len"])):
        for r in range(c["group_start"][g], c["group_start"][g + 1]):
            if only is not None and r not in only:
                continue
            P, S = int(c["prefix_len"][g]), int(c["suffix_len"][r])
            out = np.zeros((heads, hd), dtype=np.int64)
            for h in range(KVH if P + S else 0):
                K, V = [], []
                for table, n in ((c["prefix_pages"][g], P), (c["suffix_pages"][r], S)):
                    ids = table[:-(-n // PAGE)]
                    K.append(kv[h, 0][ids].reshape(-1, hd)[:n])
                    V.append(kv[h, 1][ids].reshape(-1, hd, PAGE).transpose(0, 2, 1).reshape(-1, hd)[:n])
                K, V = np.concatenate(K).astype(np.float64), np.concatenate(V).astype(np.float64)
                s = (c["q"][r, h * G:(h + 1) * G].astype(np.float64) @ K.T).astype(np.int64)      # (exact: below 2^53)
                ln2, qb, qc = (int(v) for v in c["consts"][r, h])
                x = np.minimum(s.max(1, keepdims=True) - s, 30 * ln2)
                e = ((qb - x % ln2) ** 2 + qc) >> (x // ln2)
                p = np.array([[(int(v) << 15) // int(t) for v in row] for row, t in zip(e, e.sum(1))]) if int(e.max()) >= 1 << 47 else (e << 15) // e.sum(1, keepdims=True)
                out[h * G:(h + 1) * G] = (p.astype(np.float64) @ V).astype(np.int64)
            if c["fold"] is not None:
                for h in range(heads):
                    out[h] = fold64(out[h], *c["fold"][h])
            want[r] = out
    return want


def changed_logits(x, params=None, history=(), bias=(), mask=None):
    """One row after penalties, biases (pairs) and the mask (bytes); x int32 [vocab]."""
    V = len(x)
    raw, x = x, x.astype(np.int64)
    theta, presence, frequency = (32768, 0, 0) if params is None else (int(v) for v in params)
    ids, n = np.unique(np.asarray(history, dtype=np.int64), return_counts=True)
    for v, c in zip(ids.tolist(), n.tolist()):
        if 0 <= v < V:
            y = int(x[v])
            x[v] = (y * 32768 // theta if y > 0 else -(-y * theta // 32768)) - presence - frequency * c
    for v, y in bias:
        if 0 <= v < V:
            x[v] += int(y)
    x = np.clip(x, 1 - (1 << 31), (1 << 31) - 1)
    x[raw == LOWEST] = LOWEST
    if mask is not None:
        x[np.unpackbits(mask, bitorder="little")[:V] == 0] = LOWEST
    return x


def picked(x):
    return (-2, LOWEST) if x.max() == LOWEST else (int(x.argmax()), int(x.max()))
