"""Sequences that a caller generates with the operators on its own tensors: prompts through the q/k/v site, then steps of fork, site, attention over
the paged cache, a sampled token and compaction, eagerly and as one captured graph replayed, against the definitions in whole numbers."""
import numpy as np
import pytest

from superslm_b200 import abi
from tests.support.resident import attention_rows
from tests.support.resident_more import PAGE, drawn, site_case, site_rows

pytestmark = pytest.mark.gpu
VOCAB, LAYERS, WIDTH, PAGES = 300, 2, 4, 40


@pytest.fixture()
def torch():
    t = pytest.importorskip("torch")
    assert t.cuda.is_available()
    t.cuda.set_device(0)
    return t


class Model:
    """What a token's projections are in each layer, and what the layers' attention adds to the logits."""

    def __init__(self, seed, shape, norm, halves):
        self.shape = shape
        H, KVH, hd = shape
        self.layers = [site_case(seed + i, shape, VOCAB, norm=norm, halves=halves) for i in range(LAYERS)]
        self.heads = np.random.default_rng(seed).integers(-127, 128, (LAYERS, H * hd, VOCAB)).astype(np.int64)
        self.known = {}

    def row(self, layer, token, position):
        """(q codes, constants, K codes, V codes) of a token at a position"""
        key = layer, token, position
        if key not in self.known:
            c = self.layers[layer]
            one = dict(c, wide=c["wide"][[token]], in_scales=c["in_scales"][[token]], positions=np.array([position], dtype=np.int32))
            codes, _, consts, _, K, V = site_rows(one)[0]
            self.known[key] = codes, consts, K, V
        return self.known[key]

    def logits(self, tokens):
        """of the sequence's next token"""
        H, KVH, hd = self.shape
        n, total = len(tokens), 0
        pages = -(-n // PAGE)
        for i in range(LAYERS):
            rows = [self.row(i, t, p) for p, t in enumerate(tokens)]
            kv = np.zeros((KVH, 2, pages, PAGE * hd), dtype=np.int8)
            for p, (_, _, K, V) in enumerate(rows):
                for h in range(KVH):
                    kv[h, 0, p // PAGE, p % PAGE * hd:(p % PAGE + 1) * hd] = K[h]
                    kv[h, 1, p // PAGE, p % PAGE::PAGE] = V[h]
            case = dict(q=rows[-1][0][None].astype(np.int8), consts=rows[-1][1][None], kv=kv, group_start=[0, 1], prefix_len=[0], prefix_pages=np.zeros((1, 1), dtype=np.int32),
                        suffix_len=[n], suffix_pages=np.arange(pages, dtype=np.int32)[None], fold=None)
            total = total + attention_rows(case)[0].reshape(-1) @ self.heads[i]
        return (total >> 8).astype(np.int64)


class Run:
    """The same on the GPU: `step` enqueues one step from the cache `a` back to it, over `b`."""

    def __init__(self, lib, torch, model, params, draws, parents, prompts):
        self.torch, self.model = torch, model
        H, KVH, hd = model.shape
        self.n = n = len(prompts)
        cuda = lambda x: torch.from_numpy(np.ascontiguousarray(x)).cuda()      # noqa: E731
        full = lambda *s, value=0, dtype=torch.int32: torch.full(s, value, dtype=dtype, device="cuda")      # noqa: E731
        self.kv = full(LAYERS, KVH, 2, PAGES, PAGE * hd, value=77, dtype=torch.int8)
        self.cache = [dict(holders=full(PAGES), tables=full(n, WIDTH, value=-1), lengths=full(n)) for _ in range(2)]
        self.d = [{k: cuda(v) if isinstance(v, np.ndarray) else v for k, v in c.items()} for c in model.layers]
        self.w = [cuda(h.astype(np.float64)) for h in model.heads]
        self.draws, self.parents, self.at = cuda(draws), cuda(parents), full(1, dtype=torch.int64)
        self.draw, self.parent, self.tokens = full(n), full(n), full(n)
        self.fresh = dict(drawn=full(PAGES), moves=full(n, 2), counts=full(2), status=full(n))
        self.packed = dict(new_of=full(PAGES), moves=full(PAGES // 2, 2), counts=full(2), status=full(n))
        self.refused = full(n)
        self.whole, self.nothing = cuda(np.array([0, n], dtype=np.int32)), full(1, 1)      # one group without a prefix
        a, b = self.cache
        # the prompts: every sequence goes on from itself, by as many tokens as it has
        grow = cuda(np.array([len(p) for p in prompts], dtype=np.int32))
        same = torch.arange(n, dtype=torch.int32, device="cuda")
        out = dict(out_holders=b["holders"], out_tables=b["tables"], out_lengths=b["lengths"])
        abi.Fork(lib, self.kv, **a, parents=same, grow=grow, **out, **self.fresh).run()
        tokens = cuda(np.concatenate(prompts).astype(np.int64))
        places = cuda(np.concatenate([np.arange(len(p)) for p in prompts]).astype(np.int32))
        table_of = cuda(np.concatenate([np.full(len(p), i) for i, p in enumerate(prompts)]).astype(np.int32))
        last = cuda(np.cumsum([len(p) for p in prompts]) - 1)
        codes, consts = full(len(tokens), H, hd, dtype=torch.int8), full(len(tokens), KVH, 3, dtype=torch.int64)
        logits = 0
        for i in range(LAYERS):
            self.site(lib, i, tokens, places, codes, consts, b["tables"], table_of=table_of)
            logits = logits + self.attend(lib, i, codes[last].contiguous(), consts[last].contiguous(), b)
        self.draw.copy_(self.draws[0])
        self.logits = torch.floor(logits / 256).to(torch.int32)
        self.params = cuda(np.array(params, dtype=np.int32))
        abi.Sample(lib, self.logits, self.params, self.draw, out_tokens=self.tokens, row_status=self.refused).run()
        for k in a:
            a[k].copy_(b[k])
        self.at += 1
        # a step
        self.codes, self.consts = full(n, H, hd, dtype=torch.int8), full(n, KVH, 3, dtype=torch.int64)
        self.fork = abi.Fork(lib, self.kv, **a, parents=self.parent, grow=torch.ones_like(self.parent), **out, **self.fresh)
        self.sample = abi.Sample(lib, self.logits, self.params, self.draw, out_tokens=self.tokens, row_status=self.refused)
        self.compact = abi.Compact(lib, self.kv, **b, out_holders=a["holders"], out_tables=a["tables"], **self.packed)
        self.lib = lib

    def site(self, lib, i, tokens, positions, codes, consts, tables, table_of=None):
        H, KVH, hd = self.model.shape
        d, c = self.d[i], self.model.layers[i]
        wide = d["wide"][tokens]
        q, k, v = (wide[:, x * hd:y * hd].view(-1, y - x, hd) for x, y in ((0, H), (H, H + KVH), (H + KVH, H + 2 * KVH)))
        abi.QkvSite(lib, q, k, v, d["in_scales"][tokens], positions, d["cos"], d["sin"], q_codes=codes, kv=self.kv[i], pages=tables, table_of=table_of, q_site=c["q_site"], khead=d["khead"],
                    k_landing=d["k_landing"], v_landing=d["v_landing"], q_gain=d["q_gain"], k_gain=d["k_gain"], gain_shift=c["q_shift"], k_gain_shift=c["k_shift"], halves=c["halves"],
                    consts=consts).run()

    def attend(self, lib, i, codes, consts, cache):
        """a row that is no sequence (its length is 0) has an output of zeros"""
        torch, n = self.torch, self.n
        H, KVH, hd = self.model.shape
        out = torch.zeros((n, H, hd), dtype=torch.int32, device="cuda")
        abi.PrefixAttention(lib, codes, consts, self.kv[i], self.whole, self.nothing[0], self.nothing, cache["lengths"], cache["tables"], out, max_prefix=0).run()
        return out.view(n, -1).to(torch.float64) @ self.w[i]      # (exact: below 2^53)

    def step(self):
        torch = self.torch
        a, b = self.cache
        self.draw.copy_(self.draws.index_select(0, self.at)[0])
        self.parent.copy_(self.parents.index_select(0, self.at)[0])
        fed = self.tokens.clamp(min=0).to(torch.int64)[self.parent.clamp(min=0).to(torch.int64)]
        self.fork.run()
        positions = b["lengths"] - 1
        logits = 0
        for i in range(LAYERS):
            self.site(self.lib, i, fed, positions, self.codes, self.consts, b["tables"])
            logits = logits + self.attend(self.lib, i, self.codes, self.consts, b)
        self.logits.copy_(torch.floor(logits / 256).to(torch.int32))
        self.sample.run()
        a["lengths"].copy_(b["lengths"])
        self.compact.run()
        self.at += 1


def expected(model, params, draws, parents, prompts):
    """tokens of every step (-1: no sequence)"""
    texts, out = [list(p) for p in prompts], []
    for s in range(len(draws)):
        if s > 0:
            texts = [texts[p] + [out[-1][p]] if p >= 0 and texts[p] is not None else None for p in parents[s]]
        out.append([drawn(model.logits(t), *[int(v) for v in params[i]], int(draws[s][i]))[0] if t is not None else -1 for i, t in enumerate(texts)])
    return out, texts


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("shape,norm,halves", [((4, 2, 32), "", False), ((3, 1, 64), "qk", True)])
def test_sequences_of_a_caller(gpu_lib, torch, captured, shape, norm, halves):
    model = Model(40, shape, norm, halves)
    g = np.random.default_rng(41)
    n, steps = 5, 12
    prompts = [list(g.integers(0, VOCAB, m)) for m in (3, 17, 1, 16, 30)]
    spread = model.logits(prompts[1]).std()
    params = [abi.sample_params(1.0 / spread, temperature=t, top_k=k, top_p=p, min_p=m) for t, k, p, m in ((1.0, 0, 1.0, 0.0), (0.7, 40, 0.9, 0.0), (1.5, 0, 0.8, 0.0), (1.0, 0, 1.0, 0.05), (0.0001, 1, 1.0, 0.0))]
    draws = g.integers(0, 1 << 31, (steps, n), dtype=np.int64).astype(np.int32)
    parents = np.tile(np.arange(n, dtype=np.int32), (steps, 1))
    parents[3] = 1, 1, 2, 1, 4                                # beams: one goes on three times
    parents[5] = 0, -1, 2, 3, 4                               # one ends
    parents[6] = parents[7] = 0, -1, 2, 3, 4
    parents[8] = 4, 0, 0, 3, 4                                # its place is taken
    want, texts = expected(model, params, draws, parents, prompts)
    run = Run(gpu_lib, torch, model, params, draws, parents, prompts)
    got = [run.tokens.cpu().tolist()]
    step = run.step
    if captured:
        keep = {k: v.clone() for k, v in dict(tokens=run.tokens, at=run.at, kv=run.kv).items()}, [{k: v.clone() for k, v in c.items()} for c in run.cache]
        stream = torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            run.step()                                        # (a library's first call may allocate)
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                run.step()
        torch.cuda.synchronize()
        for k, v in keep[0].items():
            getattr(run, k).copy_(v)
        for c, was in zip(run.cache, keep[1]):
            for k, v in was.items():
                c[k].copy_(v)
        step = graph.replay
    for s in range(1, steps):
        step()
        torch.cuda.synchronize()
        assert (run.fresh["status"] == 0).all() and (run.packed["status"] == 0).all() and (run.refused == 0).all()
        a = {k: v.cpu().numpy() for k, v in run.cache[0].items()}
        held = np.bincount(np.concatenate([a["tables"][i, :-(-int(m) // PAGE)] for i, m in enumerate(a["lengths"])]), minlength=PAGES)
        live = int(run.packed["counts"][1])
        assert (a["holders"] == held).all() and (held[:live] > 0).all() and (held[live:] == 0).all()
        got.append([t if m > 0 else -1 for t, m in zip(run.tokens.cpu().tolist(), a["lengths"])])
    assert got == want
    assert [len(t) if t else 0 for t in texts] == a["lengths"].tolist()
