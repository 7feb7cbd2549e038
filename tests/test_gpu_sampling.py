"""sslm_b200_seq_set_sampling: the tokens of sampled sequences are the draws from their raw logit rows (captured from the same steps) under the
definition in whole numbers, with the scale of the row that the head multiplied (from the trace of the same steps); the others of a call choose as ever."""
import ctypes as C
import dataclasses
import math

import numpy as np
import pytest

from oracle import harness as H
from superslm_b200 import abi, artifact as A
from tests.support.resident import changed_logits, picked
from tests.support.resident_more import canonical, combine, drawn

pytestmark = pytest.mark.gpu


def engine(lib, shape="tiny", cap=96, n=4, vocab=None, **model):
    shape = A.SHAPES[shape] if vocab is None else dataclasses.replace(A.SHAPES[shape], name="%s%d" % (shape, vocab), vocab=vocab)
    art = A.build_synthetic_model(shape, 0xC0, cap, **model)
    eng = abi.Engine(lib, art, blocks=n + 1, max_batch=n, max_chunk=64)
    eng.vocab, eng.art = shape.vocab, A.parse_artifact(art)
    eng.capture, eng.trace = lib.dll.sslm_b200_capture_logits, lib.dll.sslm_b200_trace
    eng.capture.argtypes, eng.trace.argtypes = [C.c_void_p, C.c_void_p], [C.c_void_p, C.c_void_p, C.c_size_t, C.POINTER(C.c_size_t)]
    eng.buf, eng.records = np.zeros(32 << 20, dtype=np.uint8), {}
    return eng


def traced(eng, f, only=None):
    """f() with its trace added to what is known (keys: position, layer, site), or what it has of one position"""
    assert eng.trace(eng.ws, eng.buf.ctypes.data, eng.buf.size, None) == 0
    try:
        return f()
    finally:
        used = C.c_size_t(0)
        assert eng.trace(eng.ws, None, 0, C.byref(used)) == 0
        eng.records.update({k: v for k, v in H.parse_trace(eng.buf[:used.value]).items() if only is None or k[0] == only})


def step(eng, seqs):
    rows = np.zeros((len(seqs), eng.vocab), dtype=np.int32)
    eng.capture(eng.ws, rows.ctypes.data)
    st, toks = traced(eng, lambda: eng.decode_step(seqs, eng.num_layers))
    eng.capture(eng.ws, None)
    assert st == 0
    return toks, rows


def row_scale(eng, position):
    """(m, e) of the row that the head multiplies: the final norm of the last layer's stream at this position"""
    _, _, codes = eng.records[(position, eng.num_layers - 1, 11)]
    h = [int(v) for v in np.frombuffer(codes, dtype=np.int8)]
    gain = eng.art.tensors(A.SEC_WEIGHTS, np.int8)["final_norm.gain"]
    root = max(1, math.isqrt((sum(v * v for v in h) << 32) // len(h)))
    top = max([1] + [abs(((v << 32) // root) * int(g)) for v, g in zip(h, gain)])
    up = 31 - top.bit_length()
    return combine(eng.art.constants(A.SEC_COMPOSITION)["final_norm"], (top << up if up >= 0 else top >> -up, -up))


def slope_of(eng, temperature, position, head=None):
    m, e = eng.art.constants(A.SEC_COMPOSITION)["embed"] if head is None else head
    m *= 127 if head is None else 1
    q, e = (m * 3098164009 << 48) // int(round(temperature * 65536)), e + 16 - 31 - 48
    while q >= 1 << 31:
        q, e = q >> 1, e + 1
    s = combine(canonical(q, e), row_scale(eng, position))
    cut = -(s[1] + 24)
    if cut < 0:
        return 1 << 30, 0
    return (s[0] >> max(0, cut - 63) if cut <= 94 else 0), min(63, cut)


def number(seed, i, given=()):
    if i < len(given):
        return given[i]
    x = (seed + (i + 1) * 0x9E3779B97F4A7C15) & (2 ** 64 - 1)
    x = (x ^ (x >> 30)) * 0xBF58476D1CE4E5B9 & (2 ** 64 - 1)
    x = (x ^ (x >> 27)) * 0x94D049BB133111EB & (2 ** 64 - 1)
    return (x ^ (x >> 31)) >> 33


def expected(eng, x, position, i, c):
    """of one row of logits as controls and masks have left it"""
    slope, cut = slope_of(eng, c.get("temperature", 1.0), position, c.get("head_scale"))
    return drawn(x.astype(np.int64).astype(np.int32), slope, cut, c.get("top_k", 0), max(1, int(c.get("top_p", 1.0) * (1 << 30))), int(c.get("min_p", 0.0) * (1 << 30)),
                 number(c.get("seed", 0), i, c.get("draws", ())))[0]


MIX = [(dict(temperature=0.7, seed=5), None), (dict(top_k=20, top_p=0.9, draws=[0, (1 << 31) - 1, 123456789]), None), (dict(temperature=1.5, min_p=0.05, seed=1 << 63), None),
       (dict(top_p=0.8, seed=9), dict(repetition=45000, presence=3000, frequency=700, biases=[(5, 40000), (9, 90000)])), (None, dict(repetition=20000, presence=-5000)), (None, None)]


@pytest.mark.parametrize("shape,vocab", [("tiny", None), ("small", None), ("mini0.5b", None), ("tiny", 40009)])
def test_tokens_are_the_draws(gpu_lib, shape, vocab):
    eng = engine(gpu_lib, shape, 96, len(MIX), vocab)
    try:
        seqs, at, produced = [], [], []
        for i, (sampling, controls) in enumerate(MIX):
            s = eng.new_seq()
            p = A.stream_uniform(10 + i, "prompt", 10 + 13 * i, 0, 40)      # (lengths that no two sequences pass through in one step)
            traced(eng, lambda: s.prefill(p, 64), len(p) - 1)
            if sampling is not None:
                s.set_sampling(**sampling)
            if controls is not None:
                s.set_controls(**controls)
            seqs.append(s)
            at.append(len(p) - 1)
            produced.append([])
        for n in range(10):
            toks, rows = step(eng, seqs)
            for i, (sampling, controls) in enumerate(MIX):
                x = rows[i].astype(np.int64)
                if controls is not None:
                    c = dict(dict(repetition=32768, presence=0, frequency=0, biases=()), **controls)
                    x = changed_logits(rows[i], (c["repetition"], c["presence"], c["frequency"]), produced[i], c["biases"])
                want = picked(x)[0] if sampling is None else expected(eng, x, at[i] + n, n, sampling)
                assert toks[i] == want, (n, i)
                produced[i].append(want)
        assert len(set(produced[0])) > 1
    finally:
        eng.close()


def test_under_a_schema(gpu_lib):
    """the mask of the sequence's state, with controls and without; the walk goes on with the token that was drawn"""
    sh = A.SHAPES["small"]
    table = A.synthetic_schemas(0xC0, sh.vocab, 2)
    eng = engine(gpu_lib, "small", 64, 3, schemas=2)
    settings = [(dict(temperature=2.0, seed=3), None), (dict(temperature=1.0, top_k=15, seed=4), dict(repetition=60000, presence=50000)), (None, None)]
    try:
        seqs, states, produced = [], [0, 0, 0], [[], [], []]
        for i, (sampling, controls) in enumerate(settings):
            h = C.c_void_p()
            assert gpu_lib.sslm_schema_lookup(eng.model, table[i % 2]["name"].encode(), C.byref(h)) == 0
            s = eng.new_seq()
            assert gpu_lib.sslm_seq_set_schema(s.handle, h) == 0
            traced(eng, lambda: s.prefill(A.stream_uniform(1 + i, "prompt", 9 + 12 * i, 0, sh.vocab - 1), 64), 8 + 12 * i)
            if sampling is not None:
                s.set_sampling(**sampling)
            if controls is not None:
                s.set_controls(**controls)
            seqs.append(s)
        for n in range(5):
            toks, rows = step(eng, seqs)
            for i, (sampling, controls) in enumerate(settings):
                row = table[i % 2]["rows"][states[i]]
                mask = np.zeros((sh.vocab + 7) // 8, dtype=np.uint8)
                for t, _ in row:
                    mask[t >> 3] |= 1 << (t & 7)
                x = changed_logits(rows[i], None if controls is None else (60000, 50000, 0), produced[i] if controls is not None else (), (), mask)
                want = expected(eng, x, 8 + 12 * i + n, n, sampling) if sampling is not None else picked(x)[0]
                assert toks[i] == want, (n, i)
                if want == -2:      # (a dead end)
                    return
                states[i] = dict(row)[want]
                produced[i].append(want)
    finally:
        eng.close()


def test_one_token_allowed_is_the_greedy_one_and_back(gpu_lib):
    art = A.build_synthetic_model("tiny", 0xC0, 96)
    eng = abi.Engine(gpu_lib, art, blocks=3, max_batch=2, max_chunk=64)
    try:
        p = A.stream_uniform(4, "prompt", 21, 0, 100)
        a, b = eng.new_seq(), eng.new_seq()
        for s in (a, b):
            s.prefill(p, 64)
        b.set_sampling(top_k=1, temperature=50.0, seed=8)
        for _ in range(3):
            st, toks = eng.decode_step([a, b], eng.num_layers)
            assert st == 0 and toks[0] == toks[1]
        b.set_sampling(temperature=None)
        for _ in range(3):
            st, toks = eng.decode_step([b, a], eng.num_layers)
            assert st == 0 and toks[0] == toks[1]
        assert a.save() == b.save()
        # sliced over several calls; the number is taken by the call that ends the token
        b.set_sampling(top_k=1, draws=[5, 6])
        assert a.decode(2, 1) == b.decode(2, 1)
    finally:
        eng.close()


def test_a_reset_begins_the_draws_again(gpu_lib):
    eng = engine(gpu_lib, "tiny", 96, 1)
    try:
        p = A.stream_uniform(6, "prompt", 12, 0, 100)
        s = eng.new_seq()
        s.set_sampling(temperature=3.0, seed=77, draws=[1 << 30])
        s.prefill(p, 64)
        first = s.decode(8, eng.num_layers)
        more = s.decode(3, eng.num_layers)
        s.reset()
        s.prefill(p, 64)
        assert s.decode(11, eng.num_layers) == first + more
        s.set_sampling(temperature=3.0, seed=78)
        s.reset()
        s.prefill(p, 64)
        assert s.decode(11, eng.num_layers) != first + more
    finally:
        eng.close()


def test_a_scale_of_the_head(gpu_lib):
    """another scale than the embedding's is another temperature"""
    eng = engine(gpu_lib, "small", 64, 1)
    try:
        m, e = eng.art.constants(A.SEC_COMPOSITION)["embed"]
        head = canonical(m * 127 >> 7, e + 7 + 2)      # about four times as coarse
        c = dict(temperature=1.2, seed=3, head_scale=head)
        s = eng.new_seq()
        traced(eng, lambda: s.prefill(A.stream_uniform(2, "prompt", 9, 0, 100), 64))
        s.set_sampling(**c)
        for n in range(4):
            toks, rows = step(eng, [s])
            assert toks[0] == expected(eng, rows[0], 8 + n, n, c)
    finally:
        eng.close()


def test_refusals(gpu_lib):
    eng = engine(gpu_lib, "tiny", 96, 1)
    bad = abi.ST["SSLM_INVALID_ARGUMENT"]
    fn = gpu_lib.dll.sslm_b200_seq_set_sampling
    fn.restype, fn.argtypes = C.c_int, [C.c_void_p, C.c_void_p]
    try:
        s = eng.new_seq()
        good = dict(struct_size=C.sizeof(abi.SslmSampling), temperature=65536, top_k=0, top_p=1 << 30, min_p=0)

        def ask(**change):
            c = abi.SslmSampling(**dict(good, **change))
            return fn(s.handle, C.addressof(c))
        assert ask() == 0
        for change in (dict(struct_size=8), dict(temperature=0), dict(temperature=-1), dict(top_k=-1), dict(top_p=0), dict(top_p=(1 << 30) + 1), dict(min_p=-1), dict(min_p=(1 << 30) + 1),
                       dict(n_draws=-1), dict(n_draws=2), dict(head_m=5), dict(head_m=1 << 31), dict(head_m=1 << 30, head_e=5000), dict(reserved=1)):
            assert ask(**change) == bad, change
        draws = (C.c_int32 * 2)(5, -1)
        assert ask(n_draws=2, draws=C.cast(draws, C.POINTER(C.c_int32))) == bad and ask(n_draws=1, draws=C.cast(draws, C.POINTER(C.c_int32))) == 0
        assert fn(None, None) == bad and fn(s.handle, None) == 0
        s.prefill(A.stream_uniform(1, "prompt", 5, 0, 100), 64)
        st, toks = eng.decode_step([s], eng.num_layers)
        assert st == 0 and toks[0] >= 0
    finally:
        eng.close()


@pytest.mark.parametrize("exchange,sampling", [(0, dict(seed=1)), (1, dict(seed=1)), (2, dict(top_k=30, seed=2))])
def test_a_wait_that_runs_out_inside_a_step(gpu_lib, exchange, sampling):
    """the sequence keeps its stream; the next step draws the token with the same number"""
    arm = gpu_lib.dll.sslm_b200_debug_withhold_exchange
    arm.argtypes = [C.c_int32, C.c_int32]
    eng = engine(gpu_lib, "tiny", 64, 1, vocab=32003)
    try:
        p = A.stream_uniform(3, "prompt", 11, 0, 100)
        s = eng.new_seq()
        s.set_sampling(**sampling)
        s.prefill(p, 64)
        want = s.decode(4, eng.num_layers)
        s.reset()
        s.prefill(p, 64)
        got = s.decode(2, eng.num_layers)
        try:
            assert arm(8, exchange) == 0
            st, _ = eng.decode_step([s], eng.num_layers)
        finally:
            arm(-1, 0)
        assert st == abi.ST["SSLM_ALLOCATION_FAILED"]
        assert got + s.decode(2, eng.num_layers) == want
    finally:
        eng.close()


@pytest.mark.parametrize("rows", [40, 300])
def test_many_rows(gpu_lib, rows):
    """one token allowed to each: what the others of the batch are given"""
    art = A.build_synthetic_model("tiny", 0xC0, 48)
    eng = abi.Engine(gpu_lib, art, blocks=rows, max_batch=rows, max_chunk=64)
    try:
        seqs = []
        for i in range(rows):
            s = eng.new_seq()
            s.prefill(A.stream_uniform(i // 2, "prompt", 4 + i // 2 % 20, 0, 100), 64)
            if i % 2:
                s.set_sampling(top_k=1, seed=i)
            seqs.append(s)
        for _ in range(3):
            st, toks = eng.decode_step(seqs, eng.num_layers)
            assert st == 0 and toks[0::2] == toks[1::2]
    finally:
        eng.close()


def test_many_rows_of_a_large_vocabulary(gpu_lib):
    """cut over one block each; few tokens of theirs have a weight"""
    rows = 72
    eng = engine(gpu_lib, n=rows, vocab=33001)
    try:
        seqs = []
        for i in range(rows):
            s = eng.new_seq()
            s.prefill(A.stream_uniform(i // 3, "prompt", 4 + i // 3 % 20, 0, 100), 64)
            if i % 3 == 1:
                s.set_sampling(top_k=1, seed=i)
            elif i % 3 == 2:
                s.set_sampling(temperature=1 / 65536, top_k=40, seed=i)      # (the second largest logit weighs nothing)
            seqs.append(s)
        for _ in range(3):
            st, toks = eng.decode_step(seqs, eng.num_layers)
            assert st == 0 and toks[0::3] == toks[1::3] == toks[2::3]
    finally:
        eng.close()


def test_a_vocabulary_that_is_too_large(gpu_lib):
    for vocab, more in ((1 << 20, 0), ((1 << 20) + 8, 1)):
        eng = engine(gpu_lib, n=1, cap=32, vocab=vocab)
        try:
            s = eng.new_seq()
            s.prefill([1, 2, 3], 64)
            if more:
                with pytest.raises(abi.SslmError):
                    s.set_sampling(top_k=1)
                continue
            st, want = eng.decode_step([s], eng.num_layers)
            s.reset()
            s.prefill([1, 2, 3], 64)
            s.set_sampling(top_k=1)
            assert st == 0 and eng.decode_step([s], eng.num_layers) == (0, want)
        finally:
            eng.close()
