"""sslm_b200_seq_set_controls: the tokens of sequences with penalties and biases are the picks of their raw logit rows (captured from the
same steps) under the definition in 64 bits; everything else of a call stays as it was."""
import ctypes as C

import numpy as np
import pytest

from superslm_b200 import abi, artifact as A
from tests.support.resident import changed_logits, picked

pytestmark = pytest.mark.gpu


@pytest.fixture()
def capture(gpu_lib):
    f = gpu_lib.dll.sslm_b200_capture_logits
    f.argtypes = [C.c_void_p, C.c_void_p]
    return lambda eng, rows: f(eng.ws, None if rows is None else rows.ctypes.data)


def engine(lib, shape="tiny", cap=96, n=4, **model):
    return abi.Engine(lib, A.build_synthetic_model(shape, 0xC0, cap, **model), blocks=n + 1, max_batch=n, max_chunk=64)


def step(eng, capture, seqs):
    """tokens and raw logit rows of one step over whole tokens"""
    V = eng.vocab
    rows = np.zeros((len(seqs), V), dtype=np.int32)
    capture(eng, rows)
    st, toks = eng.decode_step(seqs, eng.num_layers)
    capture(eng, None)
    assert st == 0
    return toks, rows


SETTINGS = [dict(repetition=45000, presence=3000, frequency=700), dict(repetition=20000, presence=-5000, frequency=0, count_given=True),
            dict(biases=[(5, 40000), (5, -1000), (9, 90000), (77, -(1 << 31))]), dict(repetition=32768, presence=1 << 30, frequency=1 << 20, count_given=True, biases=[(3, 7)])]


@pytest.mark.parametrize("shape", ["tiny", "small", "mini0.5b"])
def test_tokens_are_the_picks(gpu_lib, capture, shape):
    eng = engine(gpu_lib, shape, 96, len(SETTINGS) + 1)
    eng.vocab = A.SHAPES[shape].vocab
    try:
        seqs, given, produced = [], [], []
        for i, c in enumerate(SETTINGS + [None]):
            s = eng.new_seq()
            p = A.stream_uniform(10 + i, "prompt", 20 + 3 * i, 0, 40)
            s.prefill(p, 64)
            if c is not None:
                s.set_controls(**c)
            seqs.append(s)
            given.append([int(t) for t in p])
            produced.append([])
        for n in range(12):
            if n == 6:      # more of a prompt in between: it counts where given tokens do
                more = A.stream_uniform(50, "more", 7, 0, 40)
                for i, s in enumerate(seqs):
                    s.prefill(more, 64)
                    given[i] += [int(t) for t in more]
            toks, rows = step(eng, capture, seqs)
            for i, c in enumerate(SETTINGS + [None]):
                c = c or {}
                history = produced[i] + (given[i] if c.get("count_given") else [])
                want = changed_logits(rows[i], (c.get("repetition", 32768), c.get("presence", 0), c.get("frequency", 0)), history, c.get("biases", ()))
                if not c:
                    want = rows[i].astype(np.int64)
                assert toks[i] == picked(want)[0], (n, i)
                produced[i].append(toks[i])
        assert all(len(set(p)) > 1 for p in produced[:1])      # (the penalties do keep it from repeating itself)
    finally:
        eng.close()


def test_the_row_itself_is_the_plain_one(gpu_lib, capture):
    """a controlled sequence, and a plain one that is given the tokens it produced: the same logits at every step"""
    eng = engine(gpu_lib, "small", 64, 2)
    eng.vocab = A.SHAPES["small"].vocab
    try:
        prompt = A.stream_uniform(1, "prompt", 9, 0, eng.vocab - 1)
        a = eng.new_seq()
        a.prefill(prompt, 64)
        a.set_controls(repetition=60000, presence=20000)
        toks, rows = [], []
        for _ in range(6):
            t, r = step(eng, capture, [a])
            toks.append(t[0])
            rows.append(r[0])
        for n in range(6):
            b = eng.new_seq()
            b.prefill(np.concatenate([prompt, np.array(toks[:n], dtype=np.int32)]), 64)
            t, r = step(eng, capture, [b])
            assert (r[0] == rows[n]).all()
            b.release()
    finally:
        eng.close()


def test_the_others_of_a_batch_choose_as_ever(gpu_lib):
    n = 70
    eng = engine(gpu_lib, "tiny", 40, n)
    sh = A.SHAPES["tiny"]
    try:
        prompts = [A.stream_uniform(100 + i, "prompt", 3 + i % 9, 0, sh.vocab - 1) for i in range(n)]

        def batch(controlled):
            seqs = []
            for i, p in enumerate(prompts):
                s = eng.new_seq()
                s.prefill(p, 64)
                if i in controlled:
                    s.set_controls(biases=[(i % sh.vocab, (1 << 31) - 1)])
                seqs.append(s)
            got = [eng.decode_step(seqs, sh.layers)[1] for _ in range(4)]
            blobs = [s.save() for s in seqs]
            for s in seqs:
                s.release()
            return got, blobs
        plain, blobs = batch(())
        mixed, mixed_blobs = batch((0, 31, 69))
        for i in range(n):
            if i in (0, 31, 69):
                assert [g[i] for g in mixed] == [i] * 4      # (the bias decides)
            else:
                assert [g[i] for g in mixed] == [g[i] for g in plain] and mixed_blobs[i] == blobs[i]
    finally:
        eng.close()


@pytest.mark.parametrize("budget", [1, 2])
def test_sliced_tokens(gpu_lib, budget):
    sh = A.SHAPES["small"]
    got = []
    for b in (sh.layers, budget):
        eng = engine(gpu_lib, "small", 64, 1)
        s = eng.new_seq()
        s.prefill(A.stream_uniform(1, "prompt", 9, 0, sh.vocab - 1), 64)
        s.set_controls(repetition=50000, presence=9000, frequency=100)
        got.append(s.decode(8, b))
        eng.close()
    assert got[0] == got[1]


def test_under_a_schema(gpu_lib, capture):
    """the mask of the sequence's state and the controls together; the walk goes on with the token that was chosen"""
    sh = A.SHAPES["small"]
    table = A.synthetic_schemas(0xC0, sh.vocab, 2)
    eng = engine(gpu_lib, "small", 64, 2, schemas=2)
    eng.vocab = sh.vocab
    try:
        seqs, states, produced, controls = [], [0, 0], [[], []], []
        for i in range(2):
            h = C.c_void_p()
            assert gpu_lib.sslm_schema_lookup(eng.model, table[i]["name"].encode(), C.byref(h)) == 0
            s = eng.new_seq()
            assert gpu_lib.sslm_seq_set_schema(s.handle, h) == 0
            s.prefill(A.stream_uniform(1 + i, "prompt", 9, 0, sh.vocab - 1), 64)
            allowed = {t for t, _ in table[i]["rows"][0]}
            forbidden = next(t for t in range(sh.vocab) if t not in allowed)
            controls.append(dict(repetition=60000, presence=50000, biases=[(forbidden, (1 << 31) - 1)] + [(t, -3000 * (t % 5)) for t in sorted(allowed)[:40]]))
            s.set_controls(**controls[i])
            seqs.append(s)
        for _ in range(5):
            toks, rows = step(eng, capture, seqs)
            for i in range(2):
                row = table[i]["rows"][states[i]]
                mask = np.zeros((sh.vocab + 7) // 8, dtype=np.uint8)
                for t, _ in row:
                    mask[t >> 3] |= 1 << (t & 7)
                c = controls[i]
                want = picked(changed_logits(rows[i], (c["repetition"], c["presence"], 0), produced[i], c["biases"], mask))[0]
                assert toks[i] == want
                if want == -2:      # (a dead end)
                    return
                states[i] = dict(row)[want]
                produced[i].append(want)
    finally:
        eng.close()


def test_prefix_tokens_count_as_given(gpu_lib, capture):
    eng = engine(gpu_lib, "tiny", 64, 2)
    eng.vocab = A.SHAPES["tiny"].vocab
    try:
        pre = A.stream_uniform(3, "prefix", 25, 0, 30)
        h, c = C.c_void_p(), C.c_int32(0)
        assert gpu_lib.sslm_prefix_begin(eng.model, C.byref(eng.pool), C.byref(h)) == 0
        assert gpu_lib.sslm_prefix_prefill(eng.model, h, np.ascontiguousarray(pre, dtype=np.int32).ctypes.data_as(C.POINTER(C.c_int32)), 25, 64, 0, eng.ws, C.byref(c)) == 0
        gpu_lib.sslm_prefix_freeze(h)
        s = eng.new_seq()
        s.set_controls(repetition=60000, count_given=True, frequency=5000)
        assert gpu_lib.sslm_seq_adopt_prefix(s.handle, h) == 0
        own = A.stream_uniform(4, "own", 4, 0, 30)
        s.prefill(own, 64)
        history = [int(t) for t in pre] + [int(t) for t in own]
        for _ in range(4):
            toks, rows = step(eng, capture, [s])
            assert toks[0] == picked(changed_logits(rows[0], (60000, 0, 5000), history))[0]
            history.append(toks[0])
        # taken away, put back, reset: what counts is what the sequence has been through since
        s.set_controls(repetition=None)
        toks, rows = step(eng, capture, [s])
        assert toks[0] == int(rows[0].argmax())
        history.append(toks[0])
        s.set_controls(repetition=70000, count_given=True)
        toks, rows = step(eng, capture, [s])
        assert toks[0] == picked(changed_logits(rows[0], (70000, 0, 0), history))[0]
        s.reset()
        s.prefill(own, 64)
        toks, rows = step(eng, capture, [s])
        assert toks[0] == picked(changed_logits(rows[0], (70000, 0, 0), [int(t) for t in own]))[0]
        gpu_lib.sslm_prefix_release(h)
    finally:
        eng.close()


def test_save_blobs_and_restored_sequences(gpu_lib):
    eng = engine(gpu_lib, "tiny", 64, 3)
    sh = A.SHAPES["tiny"]
    try:
        prompt = A.stream_uniform(1, "prompt", 9, 0, sh.vocab - 1)
        a, b = eng.new_seq(), eng.new_seq()
        for s in (a, b):
            s.prefill(prompt, 64)
        a.set_controls(repetition=60000, presence=100000)
        assert a.save() == b.save()
        a.decode(2, sh.layers)
        r = abi.Sequence.restore(eng, a.save())
        a.set_controls(repetition=None)
        assert r.decode(4, sh.layers) == a.decode(4, sh.layers)
    finally:
        eng.close()


def test_a_sequence_listed_twice(gpu_lib):
    eng = engine(gpu_lib, "tiny", 64, 3)
    sh = A.SHAPES["tiny"]
    try:
        a, b = eng.new_seq(), eng.new_seq()
        for s in (a, b):
            s.prefill(A.stream_uniform(1, "prompt", 9, 0, 40), 64)
            s.set_controls(repetition=60000, presence=9000, frequency=4000, count_given=True)
        got = []
        for _ in range(4):
            st, toks = eng.decode_step([a, a], sh.layers)
            assert st == 0
            got += toks
        assert got == b.decode(8, sh.layers)
    finally:
        eng.close()


def test_a_slot_taken_again(gpu_lib):
    """controls, ids and biases end with their sequence, though the next one lies where it lay"""
    eng = abi.Engine(gpu_lib, A.build_synthetic_model("tiny", 0xC0, 64), blocks=1, max_batch=1, max_chunk=64)
    sh = A.SHAPES["tiny"]
    prompt = A.stream_uniform(1, "prompt", 9, 0, 40)

    def fresh(**controls):
        s = eng.new_seq()
        s.prefill(prompt, 64)
        if controls:
            s.set_controls(**controls)
        got = s.decode(6, sh.layers)
        s.release()
        return got
    try:
        plain, mild = fresh(), fresh(repetition=45000, count_given=True)
        assert fresh(repetition=60000, presence=1 << 28, biases=[(5, 1 << 30)]) != plain
        assert fresh() == plain and fresh(repetition=45000, count_given=True) == mild
    finally:
        eng.close()


def test_refusals(gpu_lib):
    eng = engine(gpu_lib, "tiny", 32, 1)
    sh = A.SHAPES["tiny"]
    try:
        s = eng.new_seq()
        s.prefill(A.stream_uniform(1, "prompt", 5, 0, sh.vocab - 1), 64)
        f = gpu_lib.dll.sslm_b200_seq_set_controls
        f.argtypes = [C.c_void_p, C.c_void_p]
        ints = (C.c_int32 * 1)(3)
        P = C.POINTER(C.c_int32)

        def call(**change):
            c = abi.SslmControls(struct_size=C.sizeof(abi.SslmControls), repetition=32768)
            for k, v in change.items():
                setattr(c, k, v)
            return f(s.handle, C.addressof(c))
        bad = abi.ST["SSLM_INVALID_ARGUMENT"]
        assert f(None, None) == bad
        assert call(struct_size=4) == bad and call(repetition=0) == bad and call(n_bias=-1) == bad and call(n_bias=1025) == bad
        assert call(n_bias=1) == bad and call(n_bias=1, bias_tokens=C.cast(ints, P)) == bad
        for t in (-1, sh.vocab):
            ints[0] = t
            assert call(n_bias=1, bias_tokens=C.cast(ints, P), bias_values=C.cast(ints, P)) == abi.ST["SSLM_TOKEN_ID_OUT_OF_RANGE"]
        assert s.decode(2, sh.layers) is not None      # (no controls stuck)
        assert call() == 0 and f(s.handle, None) == 0
    finally:
        eng.close()


def test_a_token_given_and_one_produced_for_every_position(gpu_lib, capture):
    """produced tokens that a prefill drops count all the same: twice as many ids as positions, biases and neighbours untouched"""
    cap = 40
    eng = engine(gpu_lib, "tiny", cap, 2)
    eng.vocab = A.SHAPES["tiny"].vocab
    try:
        a, b = eng.new_seq(), eng.new_seq()
        biases, own = [(7, 30000), (9, -20000), (11, 25000)], A.stream_uniform(3, "own", cap, 0, 60)
        for s in (a, b):
            s.set_controls(repetition=50000, presence=500, frequency=900, count_given=True, biases=biases)
        history = [[], []]
        for n in range(cap):
            for s, h in ((a, history[0]), (b, history[1])):
                s.prefill(own[n:n + 1], 64)
                h.append(int(own[n]))
            if n == cap - 1:      # (taken away and put back: all ids go to the device at once)
                a.set_controls(repetition=None)
                a.set_controls(repetition=50000, presence=500, frequency=900, count_given=True, biases=biases)
            toks, rows = step(eng, capture, [a, b])
            for i in range(2):
                assert toks[i] == picked(changed_logits(rows[i], (50000, 500, 900), history[i], biases))[0], n
                history[i].append(toks[i])
        assert len(history[0]) == 2 * cap and history[0] == history[1]
        assert eng.decode_step([a], eng.num_layers)[0] == abi.ST["SSLM_CONTEXT_CAP_EXCEEDED"]
    finally:
        eng.close()


def test_long_histories(gpu_lib, capture):
    """more ids than the table takes, and a context that is full"""
    cap = 3400
    eng = abi.Engine(gpu_lib, A.build_synthetic_model("tiny", 0xC1, cap), blocks=1, max_batch=1, max_chunk=1024)
    eng.vocab = A.SHAPES["tiny"].vocab
    try:
        s = eng.new_seq()
        p = A.stream_uniform(1, "prompt", cap - 3, 0, eng.vocab - 1)
        s.prefill(p, 1024)
        s.set_controls(repetition=40000, frequency=300, count_given=True)
        history = [int(t) for t in p]
        for _ in range(4):
            toks, rows = step(eng, capture, [s])
            assert toks[0] == picked(changed_logits(rows[0], (40000, 0, 300), history))[0]
            history.append(toks[0])
        assert eng.decode_step([s], eng.num_layers)[0] == abi.ST["SSLM_CONTEXT_CAP_EXCEEDED"]
    finally:
        eng.close()


def test_a_batch_that_grows_allocates_once(gpu_lib):
    """room for the logit rows of max_batch sequences with the first step that needs any; of all the workspace takes with the first larger one"""
    torch = pytest.importorskip("torch")
    shape = A.Shape("wide vocabulary", 128, 2, 4, 2, 32, 256, 151936)
    eng = abi.Engine(gpu_lib, A.build_synthetic_model(shape, 0xC2, 64), blocks=48, max_batch=24, max_chunk=96)
    try:
        seqs = []
        for i in range(48):
            s = eng.new_seq()
            s.prefill(A.stream_uniform(i, "prompt", 3, 0, shape.vocab - 1), 64)
            seqs.append(s)
        for s in seqs[:2]:
            assert eng.decode_step([s], shape.layers)[0] == 0      # (what kernels need to be loaded is)
        free = []
        for n in (1, 2, 3, 5, 8, 13, 24, 25, 33, 48):
            for s in seqs[:n]:
                s.set_controls(repetition=40000)
            assert eng.decode_step(seqs[:n], shape.layers)[0] == 0
            torch.cuda.synchronize()
            free.append(torch.cuda.mem_get_info()[0])
        row = shape.vocab * 4
        assert max(free[:7]) - min(free[:7]) < row
        assert max(free[7:]) - min(free[7:]) < row and 22 * row < free[6] - free[7] < 27 * row
    finally:
        eng.close()


def large_vocabulary(vocab):
    return A.Shape("v%d" % vocab, 128, 2, 4, 2, 32, 256, vocab)


@pytest.mark.parametrize("vocab", [32003, 151936])
@pytest.mark.parametrize("rows", [1, 3, 21, 64])
def test_vocabularies_that_are_cut_over_blocks(gpu_lib, capture, vocab, rows):
    """rows of several blocks: lists on both sides of where the table of names ends, a schema, and rows without controls among them"""
    shape = large_vocabulary(vocab)
    table = A.synthetic_schemas(0xC3, vocab, 2)
    eng = abi.Engine(gpu_lib, A.build_synthetic_model(shape, 0xC3, 1700, schemas=2), blocks=rows, max_batch=rows, max_chunk=1024)
    eng.vocab = vocab
    kinds = [dict(repetition=45000, presence=3000, frequency=700), dict(repetition=40000, frequency=90, count_given=True),
             dict(repetition=36000, presence=500, biases=[(7 * i % vocab, 400 * (i % 9) - 1500) for i in range(900)], count_given=True), None, "schema"]
    try:
        seqs, history, state, handles = [], [], [], []
        for name in (table[0]["name"], table[1]["name"]):
            h = C.c_void_p()
            assert gpu_lib.sslm_schema_lookup(eng.model, name.encode(), C.byref(h)) == 0
            handles.append(h)
        for i in range(rows):
            kind = kinds[i % len(kinds)] if rows > 1 else kinds[2]
            s = eng.new_seq()
            state.append(0 if kind == "schema" else None)
            if kind == "schema":
                assert gpu_lib.sslm_seq_set_schema(s.handle, handles[i % 2]) == 0
            # (1,600 ids and 900 biases are more than any table of names takes, 600 and 900 what some do)
            p = A.stream_uniform(20 + i, "prompt", 1600 if i % 15 == 2 else (600 if i % 15 == 7 else 12 + i % 30), 0, 4000)
            s.prefill(p, 1024)
            history.append([int(t) for t in p] if isinstance(kind, dict) and kind.get("count_given") else [])
            if kind == "schema":
                s.set_controls(repetition=60000, presence=20000)
            elif kind is not None:
                s.set_controls(**kind)
            seqs.append(s)
        dead = set()
        for _ in range(3):
            toks, raw = step(eng, capture, seqs)
            for i in range(rows):
                kind = kinds[i % len(kinds)] if rows > 1 else kinds[2]
                if kind is None:
                    assert toks[i] == int(raw[i].argmax())
                    continue
                mask = None
                if kind == "schema":
                    mask = np.zeros((vocab + 7) // 8, dtype=np.uint8)
                    allowed = dict(table[i % 2]["rows"][state[i]])
                    for t in allowed:
                        mask[t >> 3] |= 1 << (t & 7)
                    kind = dict(repetition=60000, presence=20000)
                want = picked(changed_logits(raw[i], (kind["repetition"], kind.get("presence", 0), kind.get("frequency", 0)), history[i], kind.get("biases", ()), mask))[0]
                assert toks[i] == want, (i, toks[i], want)
                if want == -2:
                    dead.add(i)
                    continue
                history[i].append(want)
                if state[i] is not None:
                    state[i] = allowed[want]
            if dead:      # (a dead end ends the sequence)
                break
    finally:
        eng.close()


@pytest.mark.parametrize("vocab", [32003, 151936])
def test_more_rows_than_are_cut(gpu_lib, vocab):
    """200 rows, three of them with biases that decide: the others choose as in a batch without controls"""
    shape = large_vocabulary(vocab)
    eng = abi.Engine(gpu_lib, A.build_synthetic_model(shape, 0xC4, 40), blocks=200, max_batch=200, max_chunk=64)
    try:
        seqs = []
        for i in range(200):
            s = eng.new_seq()
            s.prefill(A.stream_uniform(i, "prompt", 3 + i % 9, 0, vocab - 1), 64)
            seqs.append(s)
        def tokens(steps):
            return [eng.decode_step(seqs, shape.layers)[1] for _ in range(steps)]
        plain = tokens(3)
        for i, s in enumerate(seqs):
            s.reset()
            s.prefill(A.stream_uniform(i, "prompt", 3 + i % 9, 0, vocab - 1), 64)
        decided = {0: 5, 77: vocab - 1, 199: 16001}
        for i, t in decided.items():
            seqs[i].set_controls(biases=[(t, (1 << 31) - 1)])
        for got, want in zip(tokens(3), plain):
            assert got == [decided.get(i, t) for i, t in enumerate(want)]
    finally:
        eng.close()


@pytest.mark.parametrize("rows,exchange", [(1, 0), (1, 1), (5, 0), (5, 1), (160, 1)])
def test_a_wait_that_runs_out_inside_a_step(gpu_lib, rows, exchange):
    """the step fails, and the same step made again is right"""
    arm = gpu_lib.dll.sslm_b200_debug_withhold_exchange
    arm.argtypes = [C.c_int32, C.c_int32]
    shape = large_vocabulary(32003)
    eng = abi.Engine(gpu_lib, A.build_synthetic_model(shape, 0xC5, 40), blocks=2 * rows, max_batch=rows, max_chunk=64)
    try:
        twins = []
        for _ in range(2):
            seqs = []
            for i in range(rows):
                s = eng.new_seq()
                s.prefill(A.stream_uniform(i, "prompt", 3 + i % 9, 0, 40), 64)
                s.set_controls(repetition=60000, presence=9000, frequency=4000, count_given=True)
                seqs.append(s)
            twins.append(seqs)
        try:
            assert arm(7, exchange) == 0
            assert eng.decode_step(twins[0], shape.layers)[0] == abi.ST["SSLM_ALLOCATION_FAILED"]
        finally:
            arm(-1, 0)
        # the call ended at its first row, whose wait it was; the others were not advanced
        for _ in range(2):
            st, got = eng.decode_step(twins[0], shape.layers)
            assert st == 0 and (st, got) == eng.decode_step(twins[1], shape.layers)
    finally:
        eng.close()


@pytest.mark.parametrize("rows,exchange,budget", [(1, 1, 2), (3, 0, 2), (3, 1, 1)])
def test_a_wait_that_runs_out_between_tokens(gpu_lib, rows, exchange, budget):
    """the layers of the failed step stay done, its token is chosen by the next one: tokens, K/V and counts as if nothing had been"""
    arm = gpu_lib.dll.sslm_b200_debug_withhold_exchange
    arm.argtypes = [C.c_int32, C.c_int32]
    shape = large_vocabulary(32003)
    eng = abi.Engine(gpu_lib, A.build_synthetic_model(shape, 0xC6, 40), blocks=2 * rows, max_batch=rows, max_chunk=64)
    try:
        twins = []
        for _ in range(2):
            seqs = []
            for i in range(rows):
                s = eng.new_seq()
                s.prefill(A.stream_uniform(i, "prompt", 3 + i, 0, 40), 64)
                s.set_controls(repetition=60000, presence=9000, frequency=4000, count_given=True)
                seqs.append(s)
            twins.append(seqs)
        for seqs in twins:
            assert eng.decode_step(seqs, budget)[0] == 0
        for _ in range(shape.layers // budget - 1):
            assert [eng.decode_step(seqs, budget)[0] for seqs in twins] == [0, 0]
        try:
            assert arm(7, exchange) == 0
            assert eng.decode_step(twins[0], budget)[0] == abi.ST["SSLM_ALLOCATION_FAILED"]
        finally:
            arm(-1, 0)
        # (the first row is where it ended: the rows behind it take the failed step again)
        st, first = eng.decode_step(twins[0][:1], budget)
        assert st == 0
        rest = eng.decode_step(twins[0][1:], budget) if rows > 1 else (0, [])
        assert rest[0] == 0 and (0, first + rest[1]) == eng.decode_step(twins[1], budget)
        for _ in range(4):
            assert eng.decode_step(twins[0], budget) == eng.decode_step(twins[1], budget)
        assert [s.save() for s in twins[0]] == [s.save() for s in twins[1]]
    finally:
        eng.close()


@pytest.mark.parametrize("rows", [257, 300, 520])
def test_more_rows_than_one_launch_of_the_head_stores(gpu_lib, rows):
    """batches whose head rows run in several launches: schemas and controls on both sides of where they are cut, the others choose as ever"""
    vocab = 8191
    shape = large_vocabulary(vocab)
    table = A.synthetic_schemas(0xC7, vocab, 1)
    eng = abi.Engine(gpu_lib, A.build_synthetic_model(shape, 0xC7, 40, schemas=1), blocks=rows, max_batch=rows, max_chunk=64)
    try:
        h = C.c_void_p()
        assert gpu_lib.sslm_schema_lookup(eng.model, table[0]["name"].encode(), C.byref(h)) == 0
        bound = [3, 255, 256, rows - 1]
        decided = {0: 5, 100: vocab - 1, 254: 77, 256: sorted(t for t, _ in table[0]["rows"][0])[-1], rows - 2: 4000}
        got = []
        for controlled in (False, True):
            seqs = []
            for i in range(rows):
                s = eng.new_seq()
                if i in bound:
                    assert gpu_lib.sslm_seq_set_schema(s.handle, h) == 0
                s.prefill(A.stream_uniform(i, "prompt", 3 + i % 9, 0, vocab - 1), 64)
                if controlled and i in decided:
                    s.set_controls(biases=[(decided[i], (1 << 31) - 1)])
                seqs.append(s)
            st, toks = eng.decode_step(seqs, shape.layers)
            assert st == 0
            got.append(toks)
            for s in seqs:
                s.release()
        plain, chosen = got
        allowed = {t for t, _ in table[0]["rows"][0]}      # (a bias brings no token in that the schema leaves out)
        assert chosen == [decided[i] if i in decided and (i not in bound or decided[i] in allowed) else t for i, t in enumerate(plain)]
    finally:
        eng.close()
