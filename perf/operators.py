"""Performance cases of the operators on a caller's own tensors: the two ends of one decode step of a
batch that continues a common prompt under constraints.

  attention  integer attention of a batch of rows over the paged int8 KV pool, the rows in groups that
             share a prefix (sslm_b200_attention_prefix_resident). A row sees its group's prefix and then
             the positions of its own suffix.
  pick       penalties for repeated tokens, biases and masks on int32 logits, and the greedy token
             (sslm_b200_pick_resident).

Head counts, head dimensions and vocabularies are those of superslm_b200.artifact.SHAPES, or generic.
K, V and q are int8 codes of about normal distribution, as the requant funnel leaves them, with softmax
constants that give the attention logits a deviation of one to three. Logits are the accumulators of
an int8 vocabulary head. Everything is integers: results must be the same to the last bit.
"""
import math
import random

import numpy as np
import torch

own = False

PAGE = 16
LOWEST = -(1 << 31)


# ------------------------------------------------------------------------------------- cases
def _attention(name, shape, rows, groups, prefix, lo, hi, tokens=1, ragged=False):
    heads, kv_heads, head_dim = shape
    return dict(name=name, op="attention", heads=heads, kv_heads=kv_heads, head_dim=head_dim, rows=rows, groups=groups, prefix=prefix,
                ragged=ragged, lo=lo, hi=hi, tokens=tokens)


def listed():
    small, medium, large = (14, 2, 64), (12, 2, 128), (16, 2, 128)
    return [
        # one conversation behind a system prompt: latency is all that counts
        _attention("prefix_one_row", medium, 1, 1, 512, 37, 37),
        # a few users of the small model, a prompt that ends inside a page, replies just begun
        _attention("prefix_eight_short", small, 8, 1, 300, 1, 64),
        # a draft of four tokens each, checked in one pass: rows of one sequence share its suffix pages
        _attention("prefix_draft", small, 64, 1, 1500, 20, 200, tokens=4),
        # a busy server behind one long system prompt
        _attention("prefix_64", medium, 64, 1, 2048, 16, 256),
        # a full one, several characters with prompts of their own, one of them with none
        _attention("prefix_256_groups", medium, 256, 6, 1024, 1, 300, ragged=True),
        # questions about one long document
        _attention("prefix_long", large, 32, 1, 16384, 40, 128),
        # one conversation's next token: latency again
        dict(name="pick_one", op="pick", rows=1, vocab=151936, history=200, bias=16, mask="none", logits=False),
        # structured output: a schema's state allows about a thousand tokens
        dict(name="pick_schema", op="pick", rows=21, vocab=151936, history=512, bias=64, mask="few", logits=False),
        # a small vocabulary of odd size and histories as long as a context may be
        dict(name="pick_long_history", op="pick", rows=40, vocab=32003, history=32768, bias=300, mask="half", logits=False),
        # the processed rows are wanted too, for the caller's own sampler
        dict(name="pick_logits_out", op="pick", rows=64, vocab=151936, history=1024, bias=32, mask="half", logits=True),
        # a full server
        dict(name="pick_256", op="pick", rows=256, vocab=151936, history=1024, bias=0, mask="none", logits=False),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng: random.Random):
    if rng.random() < 0.55:
        heads, kv_heads, head_dim = rng.choice([(14, 2, 64), (12, 2, 128), (16, 2, 128), (4, 2, 32), (8, 8, 64), (6, 2, 128), (5, 1, 32), (16, 4, 64)])
        tokens = rng.choice([1, 1, 1, 2, 5])
        rows = tokens * _log_int(rng, 1, 256 // tokens)
        hi = _log_int(rng, 1, 600)
        prefix = _log_int(rng, 16, 16384)
        prefix = max(1, min(prefix, 8_000_000 // (rows * heads) - hi))
        return dict(op="attention", heads=heads, kv_heads=kv_heads, head_dim=head_dim, rows=rows, groups=rng.choice([1, 1, 2, min(8, rows)]), prefix=prefix,
                    ragged=rng.random() < 0.5, lo=rng.randint(0 if tokens == 1 else 1, hi), hi=hi, tokens=tokens)
    vocab = rng.choice([151936, _log_int(rng, 500, 151936)])
    rows = _log_int(rng, 1, 256)
    history = rng.choice([0, _log_int(rng, 1, 32768 if rows <= 64 else 2048)])
    return dict(op="pick", rows=rows, vocab=vocab, history=history, bias=rng.choice([0, _log_int(rng, 1, 1024)]), mask=rng.choice(["none", "few", "half"]),
                logits=rng.random() < 0.3)


# ------------------------------------------------------------------------------------ inputs
def _codes(shape, deviation, g):
    return (torch.randn(shape, device="cuda", generator=g) * deviation).round_().clamp_(-127, 127).to(torch.int8)


def _attention_lengths(case, seed):
    """Host-side plan of a case: rows per group, prefix lengths, suffix lengths."""
    r = np.random.default_rng([seed, 11])
    rows, groups, tokens = case["rows"], min(case["groups"], case["rows"]), case["tokens"]
    cuts = np.sort(r.choice(np.arange(1, rows), groups - 1, replace=False)) if groups > 1 else np.zeros(0, dtype=np.int64)
    start = np.concatenate([[0], cuts, [rows]]).astype(np.int32)
    if case["ragged"]:
        plen = r.integers(0, case["prefix"] + 1, groups).astype(np.int32)
        plen[0] = case["prefix"]
    else:
        plen = np.full(groups, case["prefix"], dtype=np.int32)
    base = r.integers(case["lo"], case["hi"] + 1, rows // tokens)
    slen = (base[:, None] + np.arange(tokens)[None, :]).reshape(-1).astype(np.int32)
    return start, plen, slen


def _prepare_attention(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    H, KVH, hd, rows, tokens = case["heads"], case["kv_heads"], case["head_dim"], case["rows"], case["tokens"]
    start, plen, slen = _attention_lengths(case, seed)
    groups, max_suffix = len(plen), case["hi"] + tokens - 1
    pp, sp = -(-case["prefix"] // PAGE), max(1, -(-max_suffix // PAGE))
    pages = groups * pp + rows // tokens * sp
    kv = _codes((KVH, 2, pages, PAGE * hd), 40.0, g)
    order = torch.randperm(pages, device="cuda", generator=g).to(torch.int32)
    prefix_pages = order[:groups * pp].view(groups, pp).contiguous()
    suffix_pages = order[groups * pp:].view(rows // tokens, sp).repeat_interleave(tokens, 0).contiguous()
    q = _codes((rows, H, hd), 40.0, g)
    # q . K has a deviation of 40 * 40 * sqrt(hd); a logit is that times `scale`
    spread = torch.rand((rows, KVH), device="cuda", generator=g, dtype=torch.float64) * 2 + 1
    scale = spread / (1600.0 * math.sqrt(hd))
    consts = torch.stack([torch.floor(0.6931471805599453 / scale), torch.floor(1.353 / scale), torch.floor(0.344 / 0.3585 / scale ** 2)], -1).to(torch.int64)
    fold = torch.zeros((H, 3), dtype=torch.int32, device="cuda")
    fold[:, 1] = torch.randint(1 << 30, (1 << 31) - 1, (H,), dtype=torch.int32, device="cuda", generator=g)
    fold[:, 2] = torch.randint(0, 9, (H,), dtype=torch.int32, device="cuda", generator=g)
    fold[::5, 0] = 1
    s = dict(op="attention", q=q, consts=consts, kv=kv, group_start=torch.from_numpy(start).cuda(), prefix_len=torch.from_numpy(plen).cuda(), prefix_pages=prefix_pages,
             suffix_len=torch.from_numpy(slen).cuda(), suffix_pages=suffix_pages, fold=fold, max_prefix=case["prefix"], max_suffix=max_suffix)
    if own:
        from superslm_b200 import abi, build
        s["out"] = torch.zeros((rows, H, hd), dtype=torch.int32, device="cuda")
        s["call"] = abi.PrefixAttention(abi.SslmLib(build.LIB), out=s["out"], **{k: v for k, v in s.items() if k not in ("op", "out")})
    return s


def _prepare_pick(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rows, V = case["rows"], case["vocab"]
    logits = (torch.randn((rows, V), device="cuda", generator=g) * 80000.0).to(torch.int32)

    def ids(n):      # tokens as text has them: few are frequent
        return (torch.rand((rows, n), device="cuda", generator=g) ** 3 * V).to(torch.int32).clamp_(max=V - 1)

    def lengths(n):
        v = torch.randint(n // 2, n + 1, (rows,), dtype=torch.int32, device="cuda", generator=g)
        v[0] = n
        return v
    r = np.random.default_rng([seed, 12])
    params = np.zeros((rows, 3), dtype=np.int32)
    params[:, 0] = r.integers(32768, 42599, rows)          # repetition 1.0 .. 1.3
    params[:, 1] = r.integers(-2000, 40000, rows)          # presence
    params[:, 2] = r.integers(0, 9000, rows)               # frequency
    s = dict(op="pick", logits=logits, params=torch.from_numpy(params).cuda(), history=None, history_len=None, bias_tokens=None, bias_values=None, bias_len=None,
             masks=None, mask_page=None)
    if case["history"]:
        s["history"], s["history_len"] = ids(case["history"]), lengths(case["history"])
    if case["bias"]:
        s["bias_tokens"], s["bias_len"] = ids(case["bias"]), lengths(case["bias"])
        s["bias_values"] = (torch.randn((rows, case["bias"]), device="cuda", generator=g) * 150000.0).to(torch.int32)
    if case["mask"] != "none":      # a page of bits for each of 12 states; the last one allows nothing
        share = 0.5 if case["mask"] == "half" else min(0.5, 1000.0 / V)
        bits = torch.rand((12, -(-V // 8), 8), device="cuda", generator=g) < share
        bits[11] = False
        s["masks"] = (bits.to(torch.int32) << torch.arange(8, device="cuda", dtype=torch.int32)).sum(-1).to(torch.uint8)
        s["mask_page"] = torch.from_numpy(r.integers(-1, 12, rows).astype(np.int32)).cuda()
    if own:
        from superslm_b200 import abi, build
        s["tokens"] = torch.zeros(rows, dtype=torch.int32, device="cuda")
        s["best"] = torch.zeros(rows, dtype=torch.int32, device="cuda")
        s["out"] = torch.zeros_like(logits) if case["logits"] else None
        s["call"] = abi.Pick(abi.SslmLib(build.LIB), out_tokens=s["tokens"], out_best=s["best"], out_logits=s["out"],
                             **{k: v for k, v in s.items() if k not in ("op", "tokens", "best", "out")})
    s["want_logits"] = case["logits"]
    return s


def prepare(case, seed):
    return _prepare_attention(case, seed) if case["op"] == "attention" else _prepare_pick(case, seed)


# ------------------------------------------------------------------------------- plain forms
def _plain_attention(s):
    q, kv = s["q"], s["kv"]
    rows, H, hd = q.shape
    KVH = kv.shape[0]
    G = H // KVH
    dev = q.device
    group = torch.searchsorted(s["group_start"].to(torch.int64), torch.arange(rows, device=dev), right=True) - 1
    plen = s["prefix_len"].to(torch.int64)[group]
    n = plen + s["suffix_len"]
    width = max(1, s["max_prefix"] + s["max_suffix"])
    k = torch.arange(width, device=dev)[None, :]
    shared = k < plen[:, None]
    at = torch.where(shared, k, (k - plen[:, None])).clamp_(min=0)
    from_prefix = s["prefix_pages"][group[:, None], (at // PAGE).clamp(max=s["prefix_pages"].shape[1] - 1)]
    from_suffix = torch.gather(s["suffix_pages"], 1, (at // PAGE).clamp(max=s["suffix_pages"].shape[1] - 1))
    page = torch.where(shared, from_prefix, from_suffix).to(torch.int64)
    slot = at % PAGE
    K = kv[:, 0].view(KVH, -1, PAGE, hd)[:, page, slot]                      # [KVH, rows, width, hd]
    V = kv[:, 1].view(KVH, -1, hd, PAGE).transpose(2, 3)[:, page, slot]
    Q = q.view(rows, KVH, G, hd).transpose(0, 1).float()                     # (products of int8 over at most 128 channels: exact in 32 bits)
    score = torch.matmul(Q, K.float().transpose(2, 3)).to(torch.int64)       # [KVH, rows, G, width]
    seen = (k < n[:, None])[None, :, None, :]
    top = score.masked_fill(~seen, LOWEST).amax(-1, keepdim=True)
    ln2, b, c = (s["consts"][:, :, i].t()[:, :, None, None] for i in range(3))
    x = torch.minimum((top - score).clamp_(min=0), 30 * ln2)
    z = x // ln2
    base = b - (x - z * ln2)
    e = ((base * base + c) >> z).masked_fill_(~seen, 0)
    p = (e << 15) // e.sum(-1, keepdim=True).clamp_(min=1)
    ctx = torch.matmul(p.float(), V.float()).to(torch.int64)                 # (a row's probabilities sum to 2^15 at most: exact below 2^24)
    ctx = ctx.transpose(0, 1).reshape(rows, H, hd)
    identity, mult, shift = (s["fold"][None, :, i, None].to(torch.int64) for i in range(3))
    t = ((ctx * mult + (1 << 30)) >> 31).clamp_(max=(1 << 31) - 1)
    half = torch.where(shift > 0, torch.ones_like(shift) << (shift - 1).clamp(min=0), torch.zeros_like(shift))
    folded = torch.sign(t) * ((t.abs() + half) >> shift)
    return torch.where(identity != 0, ctx, folded).to(torch.int32)


def _plain_pick(s):
    logits = s["logits"]
    rows, V = logits.shape
    dev = logits.device
    x = logits.to(torch.int64)
    allowed = logits != LOWEST
    theta, presence, frequency = (s["params"][:, i:i + 1].to(torch.int64) for i in range(3))

    def summed(tokens, lengths, values):
        inside = (torch.arange(tokens.shape[1], device=dev)[None, :] < lengths[:, None]) & (tokens >= 0) & (tokens < V)
        return torch.zeros((rows, V), dtype=torch.int64, device=dev).scatter_add_(1, tokens.to(torch.int64).clamp(0, V - 1), torch.where(inside, values, 0))
    if s["history"] is not None:
        count = summed(s["history"], s["history_len"], torch.ones((), dtype=torch.int64, device=dev))
        scaled = torch.where(x > 0, (x << 15) // theta, -((-x * theta) >> 15))
        x = torch.where(count > 0, scaled - presence - frequency * count, x)
    if s["bias_tokens"] is not None:
        x = x + summed(s["bias_tokens"], s["bias_len"], s["bias_values"].to(torch.int64))
    if s["masks"] is not None:
        v = torch.arange(V, device=dev)
        page = s["mask_page"].to(torch.int64)
        bits = (s["masks"][page.clamp(min=0)][:, v // 8] >> (v % 8).to(torch.uint8)) & 1
        allowed = allowed & ((bits != 0) | (page < 0)[:, None])
    x = torch.where(allowed, x.clamp(1 - (1 << 31), (1 << 31) - 1), LOWEST)
    best = x.amax(1)
    first = torch.where(x == best[:, None], torch.arange(V, device=dev)[None, :], V).amin(1)
    token = torch.where(best == LOWEST, -2, first)
    got = [token.to(torch.int32), best.to(torch.int32)]
    return got + [x.to(torch.int32)] if s["want_logits"] else got


def run(state):
    if own:
        state["call"].run()
        if state["op"] == "attention":
            return state["out"]
        got = [state["tokens"], state["best"]]
        return got + [state["out"]] if state["want_logits"] else got
    return _plain_attention(state) if state["op"] == "attention" else _plain_pick(state)


# -------------------------------------------------------------------------------------- work
def work(case):
    if case["op"] == "attention":
        H, KVH, hd, rows, tokens = case["heads"], case["kv_heads"], case["head_dim"], case["rows"], case["tokens"]
        groups, suffix = min(case["groups"], rows), (case["lo"] + case["hi"]) / 2 + (tokens - 1) / 2
        prefix = case["prefix"] * (0.5 + 0.5 / groups if case["ragged"] else 1.0)      # mean of the lengths
        seen, kept = rows * (prefix + suffix), groups * prefix + rows / tokens * (suffix + (tokens - 1) / 2)
        return {"bytes": 2.0 * KVH * hd * kept + 4.0 * kept / PAGE + rows * (5.0 * H * hd + 24 * KVH), "flops": 4.0 * H * hd * seen}
    rows, V = case["rows"], case["vocab"]
    listed_ids = rows * (3 * case["history"] + 6 * case["bias"])      # three quarters of the room, 4 and 8 bytes
    return {"bytes": 4.0 * rows * V * (2 if case["logits"] else 1) + listed_ids + (0 if case["mask"] == "none" else rows * 12 / 13 * V / 8), "flops": 2.0 * rows * V}


# ------------------------------------------------------------------------------- definitions
def _exact_attention(case, seed):
    s = {k: v.cpu().numpy() if torch.is_tensor(v) else v for k, v in _prepare_attention(case, seed).items() if k not in ("call", "out")}
    q, kv = s["q"].astype(np.int64), s["kv"]
    rows, H, hd = q.shape
    KVH = kv.shape[0]
    G = H // KVH
    out = np.zeros((rows, H, hd), dtype=np.int32)
    for g in range(len(s["prefix_len"])):
        P = int(s["prefix_len"][g])
        for r in range(s["group_start"][g], s["group_start"][g + 1]):
            S = int(s["suffix_len"][r])
            places = [(s["prefix_pages"][g], P), (s["suffix_pages"][r], S)]
            if P + S == 0:
                continue
            for h in range(KVH):
                K = np.concatenate([kv[h, 0][t[:-(-m // PAGE)]].reshape(-1, hd)[:m] for t, m in places]).astype(np.float64)
                V = np.concatenate([kv[h, 1][t[:-(-m // PAGE)]].reshape(-1, hd, PAGE).swapaxes(1, 2).reshape(-1, hd)[:m] for t, m in places]).astype(np.float64)
                sc = (q[r, h * G:(h + 1) * G].astype(np.float64) @ K.T).astype(np.int64)
                ln2, b, c = (int(v) for v in s["consts"][r, h])
                down = np.minimum(sc.max(1, keepdims=True) - sc, 30 * ln2)
                e = np.right_shift((b - down % ln2) ** 2 + c, down // ln2)
                p = np.left_shift(e, 15) // e.sum(1, keepdims=True)
                ctx = np.rint(p.astype(np.float64) @ V).astype(np.int64)
                for j in range(G):
                    identity, mult, shift = (int(v) for v in s["fold"][h * G + j])
                    y = ctx[j]
                    if not identity:
                        y = np.minimum((y * mult + (1 << 30)) >> 31, (1 << 31) - 1)
                        lower, rest = y >> shift, y & ((1 << shift) - 1)
                        limit = (((1 << shift) - 1) >> 1) + (y < 0)      # halves go away from zero
                        y = lower + (rest > limit)
                    out[r, h * G + j] = y
    return out


def _exact_pick(case, seed):
    s = {k: v.cpu().numpy() if torch.is_tensor(v) else v for k, v in _prepare_pick(case, seed).items() if k not in ("call", "out", "tokens", "best")}
    rows, V = s["logits"].shape
    tokens, best, out = np.zeros(rows, np.int32), np.zeros(rows, np.int32), np.zeros((rows, V), np.int32)
    for r in range(rows):
        x = s["logits"][r].astype(np.int64)
        theta, presence, frequency = (int(v) for v in s["params"][r])
        if s["history"] is not None:
            ids, n = np.unique(s["history"][r, :s["history_len"][r]], return_counts=True)
            for v, c in zip(ids.tolist(), n.tolist()):
                y = int(x[v])
                x[v] = (y * 32768 // theta if y > 0 else -(-y * theta // 32768)) - presence - frequency * c
        if s["bias_tokens"] is not None:
            for v, y in zip(s["bias_tokens"][r, :s["bias_len"][r]].tolist(), s["bias_values"][r].tolist()):
                x[v] += y
        x = np.clip(x, 1 - (1 << 31), (1 << 31) - 1)
        if s["masks"] is not None and s["mask_page"][r] >= 0:
            x[np.unpackbits(s["masks"][s["mask_page"][r]], bitorder="little")[:V] == 0] = LOWEST
        best[r], tokens[r], out[r] = x.max(), x.argmax(), x
        if best[r] == LOWEST:
            tokens[r] = -2
    return [tokens, best, out] if case["logits"] else [tokens, best]


def exact(case, seed):
    if case["op"] == "attention":
        if case["rows"] * case["heads"] * (case["prefix"] + case["hi"]) > 9_000_000:
            return None
        return _exact_attention(case, seed)
    if case["rows"] * case["history"] > 3_000_000:
        return None
    return _exact_pick(case, seed)
