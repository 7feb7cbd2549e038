"""Performance cases of the operators around attention and the pick on a caller's own tensors: what writes the cache, what moves its
pages, and what draws the next token.

  site     the q/k/v site of a layer: int32 projections of a batch of rows become rotated int8 q codes, the softmax constants of
           the row, and K and V in the pages of the int8 pool (sslm_b200_qkv_site_resident); q and K each by the row's funnel and
           a landing scale, or normed head by head
  sample   a token drawn from int32 logits with temperature, top-k, top-p and min-p and a given random number
           (sslm_b200_sample_resident)
  fork     the sequences of a paged cache continue from others, grow or end: page tables, holders, fresh pages and the copies
           of partly filled pages (sslm_b200_fork_resident)
  compact  the pages in use move to the front of the pool (sslm_b200_compact_resident)

Head counts, head dimensions, layers and vocabularies are those of superslm_b200.artifact.SHAPES, or generic. Everything is
integers: results must be the same to the last bit.
"""
import math
import random

import numpy as np
import torch

own = False

PAGE = 16
LOWEST = -(1 << 31)
Q30 = 1 << 30
# 2^-f for 0 <= f < 1, f in 32 bits behind the point, the value in 31
EXP2 = (2147483648, 1488326151, 514119776, 114090822, 14555373)
LN2_Q, B_Q, CA_Q = 744261117, 1452772687, 1030312935      # of the integer softmax: ln 2, 1.353 and 0.344 / 0.3585, 30 bits behind the point


# ------------------------------------------------------------------------------------- cases
def _site(name, shape, rows, tokens=1, norm="", rotary=0, layout="pairs", positions=4096):
    heads, kv_heads, head_dim = shape
    return dict(name=name, op="site", heads=heads, kv_heads=kv_heads, head_dim=head_dim, rows=rows, tokens=tokens, norm=norm, rotary=rotary or head_dim,
                layout=layout, positions=positions)


def _sample(name, rows, vocab, top_k=0, top_p=1.0, min_p=0.0, allowed="all", spread=2.2):
    return dict(name=name, op="sample", rows=rows, vocab=vocab, top_k=top_k, top_p=top_p, min_p=min_p, allowed=allowed, spread=spread)


def _pages(name, op, shape, sequences, longest, pages, grow=0):
    layers, kv_heads, head_dim = shape
    return dict(name=name, op=op, layers=layers, kv_heads=kv_heads, head_dim=head_dim, sequences=sequences, longest=longest, pages=pages, grow=grow)


def listed():
    medium, large = (12, 2, 128), (16, 2, 128)
    return [
        # one conversation's next token: latency is all that counts
        _site("site_one_row", medium, 1),
        # a batch of a model that norms its heads and turns half of each, in halves
        _site("site_64_normed", large, 64, norm="qk", rotary=64, layout="halves"),
        # the last chunk of a long document: rows of one sequence, one behind the other
        _site("site_prompt", medium, 8191, tokens=8191, positions=8192),
        # one conversation again
        _sample("sample_one", 1, 151936, top_k=50, top_p=0.95),
        # temperature alone
        _sample("sample_21_plain", 21, 151936),
        # structured output of a small vocabulary of odd size: a schema's state allows about a thousand tokens
        _sample("sample_40_schema", 40, 32003, top_p=0.9, allowed="few"),
        # a busy server without a limit on the number of tokens, at a temperature that spreads them
        _sample("sample_64_top_p", 64, 151936, top_p=0.9, min_p=0.001, spread=2.6),
        # a full one
        _sample("sample_256", 256, 151936, top_k=40, top_p=0.95, min_p=0.02),
        # a search of a few beams
        _pages("fork_beams", "fork", (24, 2, 64), 12, 700, 700, grow=1),
        # four answers to each of 64 questions, some of them ended
        _pages("fork_256", "fork", (28, 2, 128), 256, 320, 6000, grow=1),
        # a pool of a few sequences, and a large one after a busy hour
        _pages("compact_small", "compact", (24, 2, 64), 9, 500, 701),
        _pages("compact_large", "compact", (28, 2, 128), 200, 500, 7001),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng: random.Random):
    kind = rng.random()
    if kind < 0.3:
        shape = rng.choice([(14, 2, 64), (12, 2, 128), (16, 2, 128), (4, 2, 32), (8, 8, 64), (6, 2, 128), (5, 1, 32), (16, 4, 64)])
        rows = _log_int(rng, 1, 4000)
        c = _site("", shape, rows, tokens=rng.choice([1, rows, max(1, rows // 3)]), norm=rng.choice(["", "", "k", "qk"]),
                  rotary=rng.choice([shape[2], shape[2], shape[2] // 2]), layout=rng.choice(["pairs", "halves"]), positions=_log_int(rng, 4096, 32768))
    elif kind < 0.65:
        c = _sample("", _log_int(rng, 1, 250), rng.choice([151936, _log_int(rng, 500, 151936)]), top_k=rng.choice([0, _log_int(rng, 1, 1000)]),
                    top_p=rng.choice([1.0, round(rng.uniform(0.5, 0.98), 3)]), min_p=rng.choice([0.0, round(rng.uniform(0.0005, 0.2), 4)]),
                    allowed=rng.choice(["all", "all", "half", "few"]), spread=round(rng.uniform(1.6, 2.6), 2))
    else:
        op, shape = rng.choice(["fork", "compact"]), rng.choice([(24, 2, 64), (28, 2, 128), (5, 1, 32), (4, 8, 64)])
        longest, sequences = _log_int(rng, 20, 1500), _log_int(rng, 2, 200)
        sequences = max(2, min(sequences, 3500 * PAGE // longest))
        grow = rng.choice([0, 1, 1, 40]) if op == "fork" else 0
        c = _pages("", op, shape, sequences, longest, sequences * (3 * -(-longest // PAGE) // 2 + 2 + -(-grow // PAGE)) + rng.randint(8, 200), grow=grow)
    del c["name"]
    return c


# ------------------------------------------------------------------------------------ inputs
def _scale_of(x):
    """(m, e) with x = m 2^e and 2^30 <= m < 2^31."""
    f, e = math.frexp(x)
    m = int(round(f * (1 << 31)))
    return (m, e - 31) if m < 1 << 31 else (m >> 1, e - 30)


def _codes(shape, deviation, g):
    return (torch.randn(shape, device="cuda", generator=g) * deviation).round_().clamp_(-127, 127).to(torch.int8)


def _rotary_tables(positions, pairs, theta=1e6):
    angle = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * theta ** (-torch.arange(pairs, dtype=torch.float64, device="cuda")[None, :] / pairs)
    return (torch.cos(angle) * Q30).round().to(torch.int32), (torch.sin(angle) * Q30).round().to(torch.int32)


def _prepare_site(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = np.random.default_rng([seed, 21])
    H, KVH, hd, rows, tokens = case["heads"], case["kv_heads"], case["head_dim"], case["rows"], case["tokens"]
    # one projection's rows: q, then k, then v
    wide = (torch.randn((rows, (H + 2 * KVH) * hd), device="cuda", generator=g) * 20000.0).to(torch.int32)
    q, k, v = wide[:, :H * hd].view(rows, H, hd), wide[:, H * hd:(H + KVH) * hd].view(rows, KVH, hd), wide[:, (H + KVH) * hd:].view(rows, KVH, hd)
    in_scales = torch.zeros((rows, 2), dtype=torch.int64, device="cuda")
    in_scales[:, 0] = torch.randint(Q30, 2 * Q30, (rows,), device="cuda", generator=g)
    in_scales[:, 1] = -50
    sequences = -(-rows // tokens)
    width = -(-case["positions"] // PAGE)
    first = r.integers(0, case["positions"] - tokens + 1, sequences)
    position = (first[:, None] + np.arange(tokens)[None, :]).reshape(-1)[:rows]
    # each sequence's pages: only those that its rows touch exist
    page_of = np.repeat(np.arange(sequences), tokens)[:rows]
    touched = np.unique(page_of * width + position // PAGE)
    pages = np.full(sequences * width, -1, dtype=np.int32)
    pages[touched] = r.permutation(len(touched)).astype(np.int32)
    kv = _codes((KVH, 2, len(touched), PAGE * hd), 40.0, g)

    def landing(kind):      # a target scale for each head, and its reciprocal
        recs = []
        for _ in range(KVH):
            m, e = _scale_of(2.0 ** -19.5 * 20000.0 / 32.0 * (0.8 + 0.4 * r.random()))
            recs.append((m, e, ((1 << 62) + m // 2) // m))
        return torch.tensor(recs, dtype=torch.int64, device="cuda")
    site = _scale_of(1.0 / 127)
    khead = torch.tensor([_scale_of((1.0 + r.random()) / (1600.0 * math.sqrt(hd)) / (2.0 ** -19.5 * 80000.0 / 127)) for _ in range(KVH)], dtype=torch.int64, device="cuda")
    cos, sin = _rotary_tables(case["positions"], case["rotary"] // 2)
    gain = lambda: (torch.rand(hd, device="cuda", generator=g) * 6000 + 5000).to(torch.int16)      # noqa: E731
    s = dict(op="site", q=q, k=k, v=v, in_scales=in_scales, positions=torch.from_numpy(position.astype(np.int32)).cuda(),
             table_of=torch.from_numpy(page_of.astype(np.int32)).cuda(), pages=torch.from_numpy(pages).cuda().view(sequences, width), kv=kv, cos=cos, sin=sin,
             q_site=site, khead=khead, k_landing=landing("k"), v_landing=landing("v"), q_gain=gain() if "q" in case["norm"] else None,
             k_gain=gain() if "k" in case["norm"] else None, gain_shift=23, halves=case["layout"] == "halves", kv_heads=KVH)
    s["q_codes"] = torch.zeros((rows, H, hd), dtype=torch.int8, device="cuda")
    s["q_scales"] = torch.zeros((rows, 2), dtype=torch.int64, device="cuda")
    s["consts"] = torch.zeros((rows, KVH, 3), dtype=torch.int64, device="cuda")
    s["saturations"] = torch.zeros(rows, dtype=torch.int32, device="cuda")
    if own:
        from superslm_b200 import abi, build
        s["call"] = abi.QkvSite(abi.SslmLib(build.LIB), **{x: y for x, y in s.items() if x not in ("op", "kv_heads")})
    return s


def _prepare_sample(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = np.random.default_rng([seed, 22])
    rows, V, nat = case["rows"], case["vocab"], 36000.0
    logits = torch.randn((rows, V), device="cuda", generator=g) * (case["spread"] * nat)
    likely = torch.randint(0, V, (rows, 40), device="cuda", generator=g)      # a few tokens that the text asks for
    logits.scatter_add_(1, likely, (torch.rand((rows, 40), device="cuda", generator=g) ** 2 * 7.0 + 3.0) * nat)
    logits = logits.to(torch.int32)
    if case["allowed"] != "all":
        share = 0.5 if case["allowed"] == "half" else min(0.5, 1000.0 / V)
        logits.masked_fill_(torch.rand((rows, V), device="cuda", generator=g) >= share, LOWEST)
    params = np.zeros((rows, 5), dtype=np.int32)
    for i in range(rows):      # octaves a logit unit, in 2^-24: 1 / (temperature nat ln 2)
        m, e = _scale_of((1 << 24) / (nat * math.log(2) * (0.6 + 0.7 * r.random())))
        params[i] = m, -e, case["top_k"], max(1, int(case["top_p"] * Q30)), int(case["min_p"] * Q30)
    s = dict(op="sample", logits=logits, params=torch.from_numpy(params).cuda(), draws=torch.from_numpy(r.integers(0, 1 << 31, rows).astype(np.int32)).cuda())
    if own:
        from superslm_b200 import abi, build
        s["tokens"] = torch.zeros(rows, dtype=torch.int32, device="cuda")
        s["mass"] = torch.zeros((rows, 2), dtype=torch.int64, device="cuda")
        s["kept"] = torch.zeros(rows, dtype=torch.int32, device="cuda")
        s["call"] = abi.Sample(abi.SslmLib(build.LIB), s["logits"], s["params"], s["draws"], out_tokens=s["tokens"], out_mass=s["mass"], out_kept=s["kept"])
    return s


def _prepare_pages(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = np.random.default_rng([seed, 23])
    n, N = case["sequences"], case["pages"]
    planes, width = case["layers"] * case["kv_heads"] * 2, -(-(case["longest"] + case["grow"]) // PAGE)
    kv = torch.randint(-128, 128, (planes, N, PAGE * case["head_dim"]), dtype=torch.int8, device="cuda", generator=g)
    lengths = r.integers(case["longest"] // 3, case["longest"] + 1, n).astype(np.int32)
    lengths[0] = case["longest"]
    lengths[r.random(n) < 0.1] = 0
    # pages in use lie anywhere; every other sequence shares the full pages of the one before it
    free = iter(r.permutation(N).tolist())
    tables, holders = np.full((n, width), -1, dtype=np.int32), np.zeros(N, dtype=np.int32)
    for i in range(n):
        used = -(-int(lengths[i]) // PAGE)
        shared = int(min(lengths[i - 1], lengths[i])) // PAGE // 2 if i % 2 else 0
        tables[i, :shared] = tables[i - 1, :shared]
        tables[i, shared:used] = [next(free) for _ in range(used - shared)]
        np.add.at(holders, tables[i, :used], 1)
    s = dict(op=case["op"], kv=kv, holders=torch.from_numpy(holders).cuda(), tables=torch.from_numpy(tables).cuda(), lengths=torch.from_numpy(lengths).cuda())
    if case["op"] == "fork":      # of four neighbours the best one goes on four times, now and then; some end
        parents = np.arange(n)
        for i in range(0, n, 4):
            if r.random() < 0.6:
                parents[i:i + 4] = r.integers(i, min(n, i + 4))
        parents[r.random(n) < 0.05] = -1
        s["parents"] = torch.from_numpy(parents.astype(np.int32)).cuda()
        s["grow"] = torch.full((n,), case["grow"], dtype=torch.int32, device="cuda")
    s["out_tables"] = torch.full((n, width), -1, dtype=torch.int32, device="cuda")
    s["out_holders"] = torch.zeros(N, dtype=torch.int32, device="cuda")
    s["moves"] = torch.zeros((n if case["op"] == "fork" else N // 2, 2), dtype=torch.int32, device="cuda")
    s["counts"] = torch.zeros(2, dtype=torch.int32, device="cuda")
    if case["op"] == "fork":
        s["out_lengths"] = torch.zeros(n, dtype=torch.int32, device="cuda")
        s["drawn"] = torch.zeros(N, dtype=torch.int32, device="cuda")
        s["status"] = torch.zeros(n, dtype=torch.int32, device="cuda")
    else:
        s["new_of"] = torch.zeros(N, dtype=torch.int32, device="cuda")
    if own:
        from superslm_b200 import abi, build
        s["call"] = (abi.Fork if case["op"] == "fork" else abi.Compact)(abi.SslmLib(build.LIB), **{x: y for x, y in s.items() if x != "op"})
    return s


def prepare(case, seed):
    return {"site": _prepare_site, "sample": _prepare_sample, "fork": _prepare_pages, "compact": _prepare_pages}[case["op"]](case, seed)


# ------------------------------------------------------------------------------- plain forms
def _half_away(x, shift):
    """x / 2^shift, halves away from zero (shift >= 1)."""
    return torch.sign(x) * ((x.abs() + (1 << (shift - 1))) >> shift)


def _reciprocal(m):      # round(2^62 / m)
    return ((1 << 62) + (m >> 1)) // m


def _combined(am, ae, bm, be):
    m, e = (am * bm + (1 << 30)) >> 31, ae + be + 31
    low = m < Q30
    return torch.where(low, m << 1, m), torch.where(low, e - 1, e)


def _normed(x, gain, shift):
    """Heads of unit mean square, times the gains, as codes."""
    a = x.abs()
    top = a.amax(-1, keepdim=True)
    up = 23 - torch.floor(torch.log2(top.clamp(min=1).double())).to(torch.int64)
    y = torch.where(up >= 0, a << up.clamp(min=0), (a + (1 << (-up - 1).clamp(min=0))) >> (-up).clamp(min=0))
    mean = ((y * y).sum(-1, keepdim=True) << 6) // x.shape[-1]
    root = torch.floor(torch.sqrt(mean.double())).to(torch.int64)
    root = root - (root * root > mean).to(torch.int64)
    root = (root + ((root + 1) * (root + 1) <= mean).to(torch.int64)).clamp(min=1)
    unit = (y * ((1 << 54) // root) + (1 << 35)) >> 36
    code = (unit * gain.to(torch.int64).abs() + (1 << (shift - 1))) >> shift
    return torch.sign(x) * torch.sign(gain.to(torch.int64)) * torch.where(top > 0, code, 0)


def _landed(x, scales, landing):
    p = scales[:, 0, None, None] * landing[None, :, 2, None]
    k = 62 - (scales[:, 1, None, None] - landing[None, :, 1, None])
    a = x.abs()
    high = a * (p >> 32) + ((a * (p & 0xFFFFFFFF)) >> 32)
    return torch.sign(x) * ((high + (1 << (k - 33))) >> (k - 32))


def _rotated(x, cos, sin, halves):
    pairs = cos.shape[-1]
    turned, rest = x[..., :2 * pairs], x[..., 2 * pairs:]
    a, b = (turned[..., :pairs], turned[..., pairs:]) if halves else (turned[..., 0::2], turned[..., 1::2])
    u, v = (_half_away(t, 30).clamp(-127, 127) for t in (a * cos - b * sin, a * sin + b * cos))
    return torch.cat([u, v, rest], -1) if halves else torch.cat([torch.stack([u, v], -1).flatten(-2), rest], -1)


def _plain_site(s):
    q, k, v, scales, pos = s["q"].to(torch.int64), s["k"].to(torch.int64), s["v"].to(torch.int64), s["in_scales"], s["positions"].to(torch.int64)
    cos, sin = s["cos"][pos].to(torch.int64)[:, None, :], s["sin"][pos].to(torch.int64)[:, None, :]
    if s["q_gain"] is not None:
        codes = _normed(q, s["q_gain"], s["gain_shift"]).clamp(-127, 127)
        qm, qe = torch.full_like(scales[:, 0], s["q_site"][0]), torch.full_like(scales[:, 0], s["q_site"][1])
    else:
        top = q.abs().amax((1, 2)).clamp(min=1)
        up = 30 - torch.floor(torch.log2(top.double())).to(torch.int64)
        top = top << up
        recip = _reciprocal(top)
        p = q.abs() * recip[:, None, None]
        a = (p >> 32) * 127 + (((p & 0xFFFFFFFF) * 127) >> 32)
        cut = (30 - up)[:, None, None]
        codes = torch.sign(q) * ((a + (1 << (cut - 1).clamp(min=0))) >> cut).clamp(max=127)
        m, e = _combined(scales[:, 0], scales[:, 1], torch.full_like(top, s["q_site"][0]), torch.full_like(top, s["q_site"][1]))
        qm, qe = _combined(m, e, top, -up)
    s["q_codes"].copy_(_rotated(codes, cos, sin, s["halves"]))
    s["q_scales"].copy_(torch.stack([qm, qe], -1))
    # softmax constants: (r / 2^..) times ln 2 and 1.353, and its square times 0.9595, r the reciprocal of the combined scale
    m, e = _combined(qm[:, None], qe[:, None], s["khead"][None, :, 0], s["khead"][None, :, 1])
    r = _reciprocal(m)
    low, high, c0, c1 = r & 0xFFFFF, r >> 20, CA_Q & 0xFFFFF, CA_Q >> 20
    parts = [low * low, 2 * low * high, high * high]
    words = [parts[0] * c0, parts[1] * c0 + parts[0] * c1, parts[2] * c0 + parts[1] * c1, parts[2] * c1]
    limbs, carry = [], torch.zeros_like(r)
    for w in words + [torch.zeros_like(r)] * 4:      # (words of 20 bits of the product of up to 94)
        t = w + carry
        limbs.append(t & 0xFFFFF)
        carry = t >> 20
    limbs = torch.stack(limbs, -1)
    cut = 154 + 2 * e
    at = cut // 20
    third = sum(torch.gather(limbs, -1, (at + i).clamp(max=7)[..., None])[..., 0] << (20 * i) for i in range(3)) >> (cut - 20 * at)
    s["consts"].copy_(torch.stack([(LN2_Q * r) >> (92 + e), (B_Q * r) >> (92 + e), third], -1))
    kc = _normed(k, s["k_gain"], s["gain_shift"]) if s["k_gain"] is not None else _landed(k, scales, s["k_landing"])
    vc = _landed(v, scales, s["v_landing"])
    s["saturations"].copy_((kc.abs() > 127).sum((1, 2)) + (vc.abs() > 127).sum((1, 2)))
    kc, vc = _rotated(kc.clamp(-127, 127), cos, sin, s["halves"]), vc.clamp(-127, 127)
    rows, KVH, hd = k.shape
    page = s["pages"][s["table_of"].to(torch.int64), pos // PAGE].to(torch.int64)
    K, V = s["kv"][:, 0].view(KVH, -1, PAGE, hd), s["kv"][:, 1].view(KVH, -1, hd, PAGE)
    K[:, page, pos % PAGE] = kc.transpose(0, 1).to(torch.int8)
    V[:, page, :, pos % PAGE] = vc.to(torch.int8)
    return [s["q_codes"], s["q_scales"], s["consts"], s["saturations"], s["kv"]]


def _share(total, part, bits):      # floor(total part / 2^bits), part <= 2^bits, total < 2^62
    return (total >> bits) * part + (((total & ((1 << bits) - 1)) * part) >> bits)


def _plain_sample(s):
    x, params = s["logits"].to(torch.int64), s["params"].to(torch.int64)
    rows, V = x.shape
    slope, cut, top_k, top_p, min_p = (params[:, i:i + 1] for i in range(5))
    allowed = x != LOWEST
    top = x.amax(1, keepdim=True)
    down = torch.where(allowed, top - x, 0)
    octaves = (down * slope) >> cut
    f = (octaves & 0xFFFFFF) << 8
    p = torch.full_like(f, EXP2[4])
    for c in EXP2[3::-1]:
        p = c - ((f * p) >> 32)
    w = torch.where(allowed & (octaves < 32 << 24), p >> (octaves >> 24).clamp(max=40), 0)
    # larger logits first, then lower indices
    order = torch.sort(torch.where(allowed, down, 1 << 34), dim=1, stable=True).indices
    w = w.gather(1, order)
    rank = torch.arange(V, device=x.device)[None, :]
    w = torch.where((rank < top_k) | (top_k == 0), w, 0)
    total = w.sum(1, keepdim=True)
    before = w.cumsum(1) - w
    w = torch.where((before < _share(total, top_p, 30)) & (w >= 2 * min_p), w, 0)
    w = torch.zeros_like(w).scatter_(1, order, w)
    total = w.sum(1, keepdim=True)
    mark = _share(total, s["draws"].to(torch.int64)[:, None], 31)
    token = (w.cumsum(1) <= mark).sum(1, keepdim=True)
    any_allowed = allowed.any(1, keepdim=True)
    weight = torch.where(any_allowed, w.gather(1, token.clamp(max=V - 1)), 0)
    token = torch.where(any_allowed, token, -2)
    return [token[:, 0].to(torch.int32), torch.cat([weight, torch.where(any_allowed, total, 0)], 1), (w > 0).sum(1).to(torch.int32)]


def _plain_fork(s):
    tables, lengths, parents, holders = s["tables"].to(torch.int64), s["lengths"].to(torch.int64), s["parents"].to(torch.int64), s["holders"].to(torch.int64)
    n, width = tables.shape
    N = len(holders)
    me, at = torch.arange(n, device=tables.device), torch.arange(width, device=tables.device)[None, :]
    goes_on, moved = parents >= 0, (parents >= 0) & (parents != me)
    from_ = parents.clamp(min=0)
    before = torch.where(goes_on, lengths[from_], 0)
    after = torch.where(goes_on, before + s["grow"], 0)
    kept = torch.where(moved, before // PAGE, (before + PAGE - 1) // PAGE)      # pages that are taken over as they are
    want = (after + PAGE - 1) // PAGE - kept
    fresh = torch.sort((holders != 0).to(torch.int32), stable=True).indices      # pages that nobody holds, in order
    first = want.cumsum(0) - want
    new = fresh[(first[:, None] + at - kept[:, None]).clamp(0, N - 1)]
    is_kept, is_new = at < kept[:, None], (at >= kept[:, None]) & (at < (kept + want)[:, None])
    out = torch.where(is_kept, tables[from_], torch.where(is_new, new, s["out_tables"].to(torch.int64)))
    held = holders.clone()
    used = ((lengths + PAGE - 1) // PAGE)[:, None]
    left = (parents != me)[:, None]
    one = torch.ones((), dtype=torch.int64, device=tables.device)
    held.index_add_(0, torch.where(left & (at < used), tables, 0).flatten(), torch.where(left & (at < used), -one, 0).flatten())
    gained = (moved[:, None] & is_kept) | is_new
    held.index_add_(0, torch.where(gained, out, 0).flatten(), torch.where(gained, one, 0).flatten())
    copied = moved & (before % PAGE != 0)
    place = torch.where(copied, copied.cumsum(0) - 1, n)
    pairs = torch.stack([tables[from_].gather(1, kept[:, None].clamp(max=width - 1))[:, 0], out.gather(1, kept[:, None].clamp(max=width - 1))[:, 0]], -1)
    moves = torch.cat([s["moves"], s["moves"][:1]]).to(torch.int64).index_copy_(0, place, pairs)[:n]
    count = copied.sum()
    # (what is left of the list names its first pair, or a page with itself)
    pairs = torch.where((me < count)[:, None], moves, moves[:1] * (count > 0))
    s["kv"][:, pairs[:, 1]] = s["kv"][:, pairs[:, 0]]
    s["out_tables"].copy_(out)
    s["out_holders"].copy_(held)
    s["out_lengths"].copy_(after)
    s["drawn"].copy_(torch.where(torch.arange(N, device=tables.device) < want.sum(), fresh, s["drawn"].to(torch.int64)))
    s["moves"].copy_(torch.where((me < count)[:, None], moves, s["moves"].to(torch.int64)))
    s["counts"].copy_(torch.stack([count, want.sum()]))
    s["status"].zero_()
    return [s[x] for x in ("out_tables", "out_lengths", "out_holders", "drawn", "moves", "counts", "status", "kv")]


def _plain_compact(s):
    tables, holders = s["tables"].to(torch.int64), s["holders"].to(torch.int64)
    n, width = tables.shape
    N = len(holders)
    page = torch.arange(N, device=tables.device)
    used = holders != 0
    live = used.sum()
    hole, late = ~used & (page < live), used & (page >= live)
    count = late.sum()
    to = torch.sort((~hole).to(torch.int32), stable=True).indices[:N // 2]
    from_ = torch.sort((~late).to(torch.int32), stable=True).indices[:N // 2]
    is_move = torch.arange(N // 2, device=tables.device) < count
    new_of = torch.where(used, page, -1)
    new_of[torch.where(is_move, from_, from_[:1])] = torch.where(is_move, to, torch.where(count > 0, to[:1], new_of[from_[:1]]))
    held = torch.zeros(N + 1, dtype=torch.int64, device=tables.device).index_copy_(0, torch.where(used, new_of, N), holders)[:N]
    pairs = torch.where(is_move[:, None], torch.stack([from_, to], -1), torch.stack([from_[:1], to[:1]], -1) * (count > 0))
    for part in range(0, len(s["kv"]), 8):      # (a gather of all planes at once would hold half of the pool again)
        s["kv"][part:part + 8, pairs[:, 1]] = s["kv"][part:part + 8, pairs[:, 0]]
    listed_ = torch.arange(width, device=tables.device)[None, :] < ((s["lengths"] + PAGE - 1) // PAGE)[:, None]
    s["out_tables"].copy_(torch.where(listed_, new_of[tables.clamp(min=0)], s["out_tables"].to(torch.int64)))
    s["out_holders"].copy_(held)
    s["new_of"].copy_(new_of)
    s["moves"].copy_(torch.where(is_move[:, None], torch.stack([from_, to], -1), s["moves"].to(torch.int64)))
    s["counts"].copy_(torch.stack([count, live]))
    return [s[x] for x in ("out_tables", "out_holders", "new_of", "moves", "counts", "kv")]


def run(state):
    if own:
        state["call"].run()
        names = {"site": ("q_codes", "q_scales", "consts", "saturations", "kv"), "sample": ("tokens", "mass", "kept"),
                 "fork": ("out_tables", "out_lengths", "out_holders", "drawn", "moves", "counts", "status", "kv"),
                 "compact": ("out_tables", "out_holders", "new_of", "moves", "counts", "kv")}[state["op"]]
        return [state[x] for x in names]
    return {"site": _plain_site, "sample": _plain_sample, "fork": _plain_fork, "compact": _plain_compact}[state["op"]](state)


# -------------------------------------------------------------------------------------- work
def work(case):
    if case["op"] == "site":
        H, KVH, hd, rows = case["heads"], case["kv_heads"], case["head_dim"], case["rows"]
        tables = min(rows, case["positions"]) * case["rotary"] * 4.0      # cosines and sines of the positions
        return {"bytes": rows * (5.0 * (H + 2 * KVH) * hd + 24 * KVH + 48) + tables, "flops": 8.0 * rows * (H + KVH) * hd}
    if case["op"] == "sample":
        return {"bytes": case["rows"] * (4.0 * case["vocab"] + 48), "flops": 10.0 * case["rows"] * case["vocab"]}
    planes, page = case["layers"] * case["kv_heads"] * 2, PAGE * case["head_dim"]
    tables = 8.0 * case["sequences"] * (case["longest"] * 2 / 3) / PAGE + 8.0 * case["pages"]
    if case["op"] == "fork":      # 0.6 of the sequences continue others, and nearly all of those from inside a page
        return {"bytes": tables + 2.0 * 0.6 * 0.7 * case["sequences"] * planes * page, "flops": 1.0 * case["pages"]}
    used = min(0.9, 0.75 * 0.9 * case["sequences"] * (case["longest"] * 2 / 3 / PAGE + 0.5) / case["pages"])      # a page in use lies behind the front with 1 - used
    return {"bytes": tables + 2.0 * used * (1 - used) * case["pages"] * planes * page, "flops": 1.0 * case["pages"]}


# ------------------------------------------------------------------------------- definitions
def _host(s):
    return {k: v.cpu().numpy() if torch.is_tensor(v) else v for k, v in s.items() if k not in ("call",)}


def _exact_site(case, seed):
    s = _host(_prepare_site(case, seed))
    H, KVH, hd, rows = case["heads"], case["kv_heads"], case["head_dim"], case["rows"]
    G_bits, pairs = 30, case["rotary"] // 2

    def rounded(num, den):      # halves away from zero
        return (abs(num) * 2 + den) // (2 * den) * (1 if num >= 0 else -1)

    def clamp(x):
        return max(-127, min(127, x))

    def canonical(m, e):
        while m < 1 << 30:
            m, e = 2 * m, e - 1
        return m, e

    def combine(a, b):
        return canonical((a[0] * b[0] + (1 << 30)) >> 31, a[1] + b[1] + 31)

    def normed(x, gain):
        top = max(abs(v) for v in x)
        if top == 0:
            return [0] * len(x)
        up = 24 - top.bit_length()
        y = [v << up if up >= 0 else rounded(v, 1 << -up) for v in x]
        root = max(1, math.isqrt(sum(v * v for v in y) * 64 // len(y)))
        return [rounded(rounded(v * ((1 << 54) // root), 1 << 36) * int(g), 1 << s["gain_shift"]) for v, g in zip(y, gain)]

    def turned(x, pos):
        x = list(x)
        for i in range(pairs):
            a, b = (i, i + pairs) if s["halves"] else (2 * i, 2 * i + 1)
            c, n = int(s["cos"][pos, i]), int(s["sin"][pos, i])
            x[a], x[b] = clamp(rounded(x[a] * c - x[b] * n, 1 << G_bits)), clamp(rounded(x[a] * n + x[b] * c, 1 << G_bits))
        return x

    def landed(x, scale, rec):
        num, cut = scale[0] * rec[2], 62 - (scale[1] - rec[1])
        return [rounded(v * num, 1 << cut) for v in x]
    for r in range(rows):
        q, k, v = ([[int(t) for t in head] for head in s[x][r]] for x in "qkv")
        scale, pos = [int(t) for t in s["in_scales"][r]], int(s["positions"][r])
        if s["q_gain"] is not None:
            codes, out = [normed(x, s["q_gain"]) for x in q], s["q_site"]
        else:
            top = max(1, max(abs(t) for x in q for t in x))
            up = 31 - top.bit_length()
            recip = ((1 << 62) + (top << up) // 2) // (top << up)
            codes = [[min(127, (abs(t) * recip * 127 + (1 << (61 - up))) >> (62 - up)) * (1 if t > 0 else -1) for t in x] for x in q]
            out = combine(combine(scale, s["q_site"]), (top << up, -up))
        s["q_codes"][r] = [turned([clamp(t) for t in x], pos) for x in codes]
        s["q_scales"][r] = out
        sat = 0
        page = int(s["pages"][s["table_of"][r], pos // PAGE])
        for h in range(KVH):
            m, e = combine(out, [int(t) for t in s["khead"][h]])
            recip = ((1 << 62) + m // 2) // m
            s["consts"][r, h] = LN2_Q * recip >> (92 + e), B_Q * recip >> (92 + e), recip * recip * CA_Q >> (154 + 2 * e)
            kc = normed(k[h], s["k_gain"]) if s["k_gain"] is not None else landed(k[h], scale, [int(t) for t in s["k_landing"][h]])
            vc = landed(v[h], scale, [int(t) for t in s["v_landing"][h]])
            sat += sum(abs(t) > 127 for t in kc + vc)
            s["kv"][h, 0, page].reshape(PAGE, hd)[pos % PAGE] = turned([clamp(t) for t in kc], pos)
            s["kv"][h, 1, page].reshape(hd, PAGE)[:, pos % PAGE] = [clamp(t) for t in vc]
        s["saturations"][r] = sat
    return [s[x] for x in ("q_codes", "q_scales", "consts", "saturations", "kv")]


def _exact_sample(case, seed):
    s = _host(_prepare_sample(case, seed))
    rows, V = s["logits"].shape
    tokens, mass, kept = np.zeros(rows, np.int32), np.zeros((rows, 2), np.int64), np.zeros(rows, np.int32)
    for r in range(rows):
        x = s["logits"][r].astype(np.int64)
        slope, cut, top_k, top_p, min_p = (int(t) for t in s["params"][r])
        ids = np.flatnonzero(x != LOWEST)
        if len(ids) == 0:
            tokens[r] = -2
            continue
        ids = ids[np.lexsort((ids, -x[ids]))]
        t = (x[ids[0]] - x[ids]) * slope >> cut
        ids, t = ids[t < 32 << 24], t[t < 32 << 24]
        if top_k:
            ids, t = ids[:top_k], t[:top_k]
        f = (t % (1 << 24)).astype(np.uint64) << np.uint64(8)
        w = np.full(len(t), EXP2[4], np.uint64)
        for c in (3, 2, 1, 0):
            w = np.uint64(EXP2[c]) - (f * w >> np.uint64(32))
        w = (w >> (t >> 24).astype(np.uint64)).astype(np.int64)
        enough = int(w.sum()) * top_p >> 30
        keep = (np.cumsum(w) - w < enough) & (w >= 2 * min_p) & (w > 0)
        ids, w = ids[keep], w[keep]
        back = np.argsort(ids)
        ids, w = ids[back], w[back]
        total = int(w.sum())
        at = int(np.searchsorted(np.cumsum(w), total * int(s["draws"][r]) >> 31, side="right"))
        tokens[r], mass[r], kept[r] = ids[at], (w[at], total), len(ids)
    return [tokens, mass, kept]


def _exact_fork(case, seed):
    s = _host(_prepare_pages(case, seed))
    free = [p for p in range(len(s["holders"])) if s["holders"][p] == 0]
    held = s["holders"].copy()
    copies, taken = [], 0
    for i, parent in enumerate(s["parents"].tolist()):
        old = s["tables"][i, :-(-int(s["lengths"][i]) // PAGE)].tolist()
        if parent < 0:
            s["out_lengths"][i] = 0
        else:
            length = int(s["lengths"][parent])
            pages = s["tables"][parent, :length // PAGE if parent != i else -(-length // PAGE)].tolist()
            s["out_lengths"][i] = length + s["grow"][i]
            if parent != i:
                for p in pages:
                    held[p] += 1
                if length % PAGE:
                    copies.append((int(s["tables"][parent, length // PAGE]), free[taken]))
            while len(pages) * PAGE < s["out_lengths"][i]:
                pages.append(free[taken])
                held[free[taken]] += 1
                taken += 1
            s["out_tables"][i, :len(pages)] = pages
        if parent != i:
            for p in old:
                held[p] -= 1
    for j, (a, b) in enumerate(copies):
        s["kv"][:, b] = s["kv"][:, a]
        s["moves"][j] = a, b
    s["out_holders"], s["counts"] = held, np.array([len(copies), taken], np.int32)
    s["drawn"][:taken] = free[:taken]
    return [s[x] for x in ("out_tables", "out_lengths", "out_holders", "drawn", "moves", "counts", "status", "kv")]


def _exact_compact(case, seed):
    s = _host(_prepare_pages(case, seed))
    used = [p for p in range(len(s["holders"])) if s["holders"][p]]
    live = len(used)
    holes = [p for p in range(live) if not s["holders"][p]]
    new = {p: p for p in used if p < live}
    new.update(zip([p for p in used if p >= live], holes))
    s["new_of"][:] = -1
    for j, (a, b) in enumerate((a, b) for a, b in new.items() if a != b):
        s["moves"][j] = a, b
        s["kv"][:, b] = s["kv"][:, a]
    for a, b in new.items():
        s["new_of"][a], s["out_holders"][b] = b, s["holders"][a]
    for i in range(len(s["tables"])):
        for j in range(-(-int(s["lengths"][i]) // PAGE)):
            s["out_tables"][i, j] = new[int(s["tables"][i, j])]
    s["counts"][:] = len(holes), live
    return [s[x] for x in ("out_tables", "out_holders", "new_of", "moves", "counts", "kv")]


def exact(case, seed):
    if case["op"] == "site":
        return None if case["rows"] * (case["heads"] + 2 * case["kv_heads"]) * case["head_dim"] > 400_000 else _exact_site(case, seed)
    if case["op"] == "sample":
        return _exact_sample(case, seed)
    if case["layers"] * case["kv_heads"] * 2 * case["pages"] * PAGE * case["head_dim"] > 200_000_000:
        return None
    return _exact_fork(case, seed) if case["op"] == "fork" else _exact_compact(case, seed)
