"""Decode rows whose sequences adopted one prefix, attended together (sslm_b200_set_prefix_attention): the same tokens, K/V, scales and
counters as row by row, whatever else is in the batch."""
import ctypes as C

import numpy as np
import pytest

from superslm_b200 import abi, artifact as A

pytestmark = pytest.mark.gpu


@pytest.fixture()
def dll(gpu_lib):
    d = gpu_lib.dll
    d.sslm_b200_prefix_attention_launches.restype = C.c_uint64
    yield d
    d.sslm_b200_set_prefix_attention(1)
    d.sslm_b200_set_attention_splits(0)


class Prefix:
    def __init__(self, eng, tokens):
        self.eng, self.h = eng, C.c_void_p()
        assert eng.lib.sslm_prefix_begin(eng.model, C.byref(eng.pool), C.byref(self.h)) == 0
        toks, done = np.ascontiguousarray(tokens, dtype=np.int32), 0
        while done < len(toks):
            c = C.c_int32(0)
            assert eng.lib.sslm_prefix_prefill(eng.model, self.h, toks[done:].ctypes.data_as(C.POINTER(C.c_int32)), len(toks) - done, 128, 0, eng.ws, C.byref(c)) == 0
            done += c.value
        assert eng.lib.sslm_prefix_freeze(self.h) == 0

    def adopt(self):
        s = self.eng.new_seq()
        assert self.eng.lib.sslm_seq_adopt_prefix(s.handle, self.h) == 0
        return s

    def release(self):
        assert self.eng.lib.sslm_prefix_release(self.h) == 0


def run(dll, lib, shape, mode, prefixes, members, steps=3, budget=None, splits=0, adapted=(), twice=(), **model):
    """members: (prefix number or None, tokens of its own) per sequence. adapted: which of them have an adapter, in turn one of
    two; twice: which are listed a second time at the end of the batch. Tokens of every step and the save blobs."""
    dll.sslm_b200_set_prefix_attention(mode)
    dll.sslm_b200_set_attention_splits(splits)
    sh = A.SHAPES[shape]
    cap = max((prefixes[p] if p is not None else 0) + n for p, n in members) + steps + 2
    cap += steps if twice else 0
    art = A.build_synthetic_model(shape, 0x5A17, cap, **model)
    eng = abi.Engine(lib, art, blocks=len(members) + len(prefixes), max_batch=len(members), max_chunk=128)
    try:
        pf = [Prefix(eng, A.stream_uniform(0x900 + i, "prefix", n, 0, sh.vocab - 1)) for i, n in enumerate(prefixes)]
        seqs = []
        for i, (p, n) in enumerate(members):
            s = pf[p].adopt() if p is not None else eng.new_seq()
            if n:
                s.prefill(A.stream_uniform(0x500 + i, "own", n, 0, sh.vocab - 1), 128)
            seqs.append(s)
        adapters = [eng.map_adapter(A.build_synthetic_adapter(art, 0x77 + i, 16 * (i + 1))) for i in range(2 if adapted else 0)]
        for i in adapted:
            seqs[i].set_adapter(adapters[i % 2])
        for p in pf:
            p.release()
        before = dll.sslm_b200_prefix_attention_launches()
        tokens = []
        for _ in range(steps * (1 if budget is None else -(-sh.layers // budget)) + 1):
            st, got = eng.decode_step(seqs + [seqs[i] for i in twice], budget or sh.layers)
            assert st == 0
            tokens.append(got)
        return tokens, [s.save() for s in seqs], dll.sslm_b200_prefix_attention_launches() - before
    finally:
        eng.close()


MIXES = {
    "one": ([100], [(0, i % 7) for i in range(9)]),
    "two and others": ([64, 333], [(0, 3), (None, 20), (1, 0), (1, 30), (0, 1), (None, 90), (1, 17), (None, 1), (0, 40)]),
    "pairs": ([16, 48, 33], [(0, 1), (1, 2), (2, 5), (0, 9), (1, 1), (2, 40)]),
    "a lone one": ([80, 50], [(0, 2), (0, 3), (1, 4), (None, 11)]),
    "less than a page": ([9, 40], [(0, 2), (0, 3), (1, 4), (1, 1)]),
}


@pytest.mark.parametrize("shape", ["tiny", "small", "mini1.5b", "mini0.5b"])
@pytest.mark.parametrize("mix", sorted(MIXES))
def test_together_and_apart(dll, gpu_lib, shape, mix):
    prefixes, members = MIXES[mix]
    apart = run(dll, gpu_lib, shape, 0, prefixes, members)
    together = run(dll, gpu_lib, shape, 2, prefixes, members)
    assert apart[2] == 0 and together[2] > 0
    assert together[0] == apart[0]
    assert together[1] == apart[1]


@pytest.mark.parametrize("splits", [1, 2, 4, 8, 16])
def test_every_cut(dll, gpu_lib, splits):
    prefixes, members = [700, 20], [(0, 1 + 13 * i) for i in range(6)] + [(1, 9), (1, 60), (None, 200)]
    apart = run(dll, gpu_lib, "mini1.5b", 0, prefixes, members)
    together = run(dll, gpu_lib, "mini1.5b", 2, prefixes, members, splits=splits)
    assert together[2] > 0 and together[:2] == apart[:2]


@pytest.mark.parametrize("budget", [1, 2])
def test_sliced_tokens(dll, gpu_lib, budget):
    prefixes, members = [90], [(0, 1 + i) for i in range(5)] + [(None, 7)]
    apart = run(dll, gpu_lib, "small", 0, prefixes, members, budget=budget)
    together = run(dll, gpu_lib, "small", 2, prefixes, members, budget=budget)
    assert together[2] > 0 and together[:2] == apart[:2]


def test_biased_projections(dll, gpu_lib):
    prefixes, members = [120], [(0, 1 + 5 * i) for i in range(7)]
    apart = run(dll, gpu_lib, "tiny", 0, prefixes, members, bias_bits=28)
    together = run(dll, gpu_lib, "tiny", 2, prefixes, members, bias_bits=28)
    assert together[2] > 0 and together[:2] == apart[:2]


@pytest.mark.parametrize("shape", ["small", "mini0.5b"])
def test_adapters_beside_it(dll, gpu_lib, shape):
    prefixes, members = [120, 33], [(i % 2, 1 + 5 * i) for i in range(8)] + [(None, 9), (None, 30)]
    apart = run(dll, gpu_lib, shape, 0, prefixes, members, adapted=(0, 3, 4, 7, 8))
    together = run(dll, gpu_lib, shape, 2, prefixes, members, adapted=(0, 3, 4, 7, 8))
    assert together[2] > 0 and together[:2] == apart[:2]


def test_sequences_listed_twice(dll, gpu_lib):
    prefixes, members = [70], [(0, 1 + 5 * i) for i in range(5)] + [(None, 9)]
    apart = run(dll, gpu_lib, "small", 0, prefixes, members, twice=(0, 2, 5))
    together = run(dll, gpu_lib, "small", 2, prefixes, members, twice=(0, 2, 5))
    assert together[2] > 0 and together[:2] == apart[:2]


def test_where_it_is_chosen(dll, gpu_lib):
    """mode 1: many rows behind a long prefix, not few or short ones"""
    many, few, short = ([1536], [(0, 1 + i % 5) for i in range(40)]), ([1536], [(0, 1 + i) for i in range(4)]), ([64], [(0, 1 + i % 5) for i in range(40)])
    assert run(dll, gpu_lib, "tiny", 1, *many, steps=1)[2] > 0
    assert run(dll, gpu_lib, "tiny", 1, *few, steps=1)[2] == 0
    assert run(dll, gpu_lib, "tiny", 1, *short, steps=1)[2] == 0


def test_sequences_that_left_their_prefix(dll, gpu_lib):
    """reset, re-adopted and restored sequences share what they hold now, not what they held"""
    dll.sslm_b200_set_prefix_attention(2)
    sh = A.SHAPES["small"]
    eng = abi.Engine(gpu_lib, A.build_synthetic_model("small", 3, 260), blocks=12, max_batch=8, max_chunk=128)
    try:
        own = [A.stream_uniform(60 + i, "own", 5 + i, 0, sh.vocab - 1) for i in range(4)]
        pre = [A.stream_uniform(70 + i, "prefix", 100, 0, sh.vocab - 1) for i in range(2)]
        pf = [Prefix(eng, p) for p in pre]

        def fresh(prompt):
            s = eng.new_seq()
            s.prefill(prompt, 128)
            return s
        a, b, c, d = (pf[0].adopt() for _ in range(4))
        b.reset()
        b.prefill(own[1], 128)                                  # shares nothing any more
        c.reset()
        assert eng.lib.sslm_seq_adopt_prefix(c.handle, pf[1].h) == 0
        c.prefill(own[2], 128)
        a.prefill(own[0], 128)
        d.prefill(own[3], 128)
        got = [eng.decode_step([a, b, c, d], sh.layers)[1]]
        e = abi.Sequence.restore(eng, d.save())                 # holds copies
        before = dll.sslm_b200_prefix_attention_launches()
        got += [eng.decode_step([a, b, c, d, e], sh.layers)[1] for _ in range(3)]
        assert dll.sslm_b200_prefix_attention_launches() - before == 3 * sh.layers      # (a and d)
        dll.sslm_b200_set_prefix_attention(0)
        plain = [fresh(p) for p in (np.concatenate([pre[0], own[0]]), own[1], np.concatenate([pre[1], own[2]]), np.concatenate([pre[0], own[3]]))]
        want = [eng.decode_step(plain, sh.layers)[1] for _ in range(4)]
        assert [g[:4] for g in got] == want and [g[4] for g in got[1:]] == [w[3] for w in want[1:]]
    finally:
        eng.close()


def test_a_wait_that_runs_out_inside_a_step(dll, gpu_lib):
    """the step fails like any refused one, and the next one is right"""
    dll.sslm_b200_set_prefix_attention(2)
    dll.sslm_b200_set_attention_splits(4)
    arm = dll.sslm_b200_debug_withhold_exchange
    arm.argtypes = [C.c_int32, C.c_int32]
    sh = A.SHAPES["mini1.5b"]
    eng = abi.Engine(gpu_lib, A.build_synthetic_model("mini1.5b", 4, 700), blocks=5, max_batch=4, max_chunk=512)
    try:
        pf = Prefix(eng, A.stream_uniform(1, "prefix", 600, 0, sh.vocab - 1))
        seqs = [pf.adopt() for _ in range(3)]
        for i, s in enumerate(seqs):
            s.prefill(A.stream_uniform(2 + i, "own", 3 + i, 0, sh.vocab - 1), 128)
        twin = pf.adopt()
        twin.prefill(A.stream_uniform(2, "own", 3, 0, sh.vocab - 1), 128)
        assert eng.decode_step(seqs, sh.layers)[0] == 0
        for exchange in range(4):
            try:
                assert arm(6, exchange) == 0
                assert eng.decode_step(seqs, sh.layers)[0] == abi.ST["SSLM_ALLOCATION_FAILED"]
            finally:
                arm(-1, 0)
        st, got = eng.decode_step(seqs, sh.layers)
        assert st == 0
        dll.sslm_b200_set_prefix_attention(0)
        assert twin.decode(2, sh.layers)[1] == got[0]
    finally:
        eng.close()


@pytest.mark.parametrize("prefixes,members,chosen", [
    ([1024], [(0, 1 + i % 7) for i in range(64)], True),                                                    # many rows behind one prefix
    ([1024], [(0, 1 + i % 7) for i in range(64)] + [(None, 20 + i) for i in range(4)], False),              # the same beside four others
    ([2048], [(0, 1 + i % 7) for i in range(12)], False),                                                   # few rows
    ([4096], [(0, 1 + i) for i in range(4)], False),
    ([4096], [(0, 1 + i) for i in range(8)], True),
    ([1024] * 32, [(i % 32, 1 + i % 5) for i in range(128)], False),                                        # many small groups
    ([1024], [(0, 300 + 20 * (i % 5)) for i in range(64)], False),                                          # suffixes that are not short
    ([2048, 128], [(0, 1 + i % 7) for i in range(40)] + [(1, 1 + i % 7) for i in range(4)], True),          # alike enough to be cut together
    ([8192, 64], [(0, 1), (0, 2)] + [(1, 1 + i % 7) for i in range(30)], False),                            # a long prefix of few, a short one of many
    ([8192, 64], [(0, 1 + i) for i in range(30)] + [(1, 1 + i % 7) for i in range(30)], True)])
def test_where_it_is_the_faster_one(dll, gpu_lib, prefixes, members, chosen):
    """mode 1 takes what was measured to gain, and leaves what was measured to lose"""
    got = run(dll, gpu_lib, "tiny", 1, prefixes, members, steps=1)
    assert (got[2] > 0) == chosen


@pytest.mark.parametrize("shape", ["tiny", "mini0.5b"])
def test_where_it_is_chosen_the_outputs_are_the_same(dll, gpu_lib, shape):
    """the default mode, with as many rows as it wants and groups that it leaves out"""
    prefixes, members = [1040, 80], [(0, 1 + i % 7) for i in range(70)]
    apart, chosen = (run(dll, gpu_lib, shape, mode, prefixes, members, steps=2) for mode in (0, 1))
    assert apart[2] == 0 and chosen[2] > 0 and chosen[:2] == apart[:2]


def test_groups_that_are_left_out(dll, gpu_lib):
    """short groups stay with the others where long ones are attended together without them"""
    prefixes, members = [4096, 64], [(0, 1 + i % 7) for i in range(36)] + [(1, 1 + i % 5) for i in range(60)] + [(None, 1 + i % 9) for i in range(10)]
    apart, chosen = (run(dll, gpu_lib, "tiny", mode, prefixes, members, steps=2) for mode in (0, 1))
    assert apart[2] == 0 and chosen[2] > 0 and chosen[:2] == apart[:2]


@pytest.mark.parametrize("mode", [1, 2])
def test_sequences_at_different_layers(dll, gpu_lib, mode):
    """rows that start on several layers share in parts of their own, each with its groups"""
    sh = A.SHAPES["small"]
    length = 1040 if mode == 1 else 90
    each = 66 if mode == 1 else 4
    got = []
    for m in (0, mode):
        dll.sslm_b200_set_prefix_attention(m)
        eng = abi.Engine(gpu_lib, A.build_synthetic_model("small", 5, length + 60), blocks=3 * each + 6, max_batch=3 * each, max_chunk=256)
        try:
            pf = [Prefix(eng, A.stream_uniform(80 + i, "prefix", n, 0, sh.vocab - 1)) for i, n in enumerate((length, 40))]
            seqs = []
            for i in range(3 * each):
                s = pf[0 if mode == 1 or i % 4 < 3 else 1].adopt() if i % 9 != 8 or mode == 1 else eng.new_seq()
                s.prefill(A.stream_uniform(90 + i, "own", 1 + i % 5, 0, sh.vocab - 1), 128)
                seqs.append(s)
            assert eng.decode_step(seqs, sh.layers)[0] == 0                    # (the token that the prompt leaves)
            assert eng.decode_step(seqs[:2 * each], 1)[0] == 0                 # two thirds are a layer on
            assert eng.decode_step(seqs[:each], 1)[0] == 0                     # one third two
            before = dll.sslm_b200_prefix_attention_launches()
            tokens = []
            order = np.random.default_rng(3).permutation(len(seqs))
            for _ in range(2 * sh.layers):
                st, t = eng.decode_step([seqs[i] for i in order], 1)
                assert st == 0
                tokens.append(t)
            launches = dll.sslm_b200_prefix_attention_launches() - before
            assert launches == (0 if m == 0 else 2 * sh.layers * sh.layers)    # (a part for each layer that rows start on)
            got.append((tokens, [s.save() for s in seqs]))
            for p in pf:
                p.release()
        finally:
            eng.close()
    assert got[0] == got[1]
