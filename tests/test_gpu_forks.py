"""sslm_b200_seq_fork: a sequence that goes on from where another one is, as if it had been given all that was before."""
import ctypes as C

import pytest

from superslm_b200 import abi, artifact as A

pytestmark = pytest.mark.gpu


def engine(lib, shape="small", cap=128, blocks=6, **model):
    return abi.Engine(lib, A.build_synthetic_model(shape, 0xF0, cap, **model), blocks=blocks, max_batch=blocks, max_chunk=64)


@pytest.mark.parametrize("shape", ["tiny", "small", "mini1.5b"])
@pytest.mark.parametrize("length,made", [(0, 0), (1, 0), (15, 0), (16, 0), (17, 3), (32, 0), (30, 2), (40, 9)])
def test_child_equals_a_sequence_that_was_given_everything(gpu_lib, shape, length, made):
    eng = engine(gpu_lib, shape)
    try:
        p = A.stream_uniform(length, "prompt", length, 0, 100) if length else []
        more = A.stream_uniform(7, "more", 5, 0, 100)
        parent, plain = eng.new_seq(), eng.new_seq()
        for s in (parent, plain):
            if length:
                s.prefill(p, 64)
                s.decode(made, eng.num_layers)
        child = parent.fork()
        if length:
            assert child.save() == plain.save() == parent.save()
        for s in (child, plain):
            s.prefill(more, 64)
        assert child.decode(20, eng.num_layers) == plain.decode(20, eng.num_layers)
        assert child.save() == plain.save()
        # the parent goes on as if nothing had been
        plain.reset()
        if length:
            plain.prefill(p, 64)
            plain.decode(made, eng.num_layers)
            assert parent.decode(20, eng.num_layers) == plain.decode(20, eng.num_layers) and parent.save() == plain.save()
    finally:
        eng.close()


def test_branches_of_branches(gpu_lib):
    """of every length, in one batch and by themselves; parents that end first; sequences that were something else"""
    eng = engine(gpu_lib, "small", 128, 9)
    try:
        p = A.stream_uniform(1, "prompt", 33, 0, 100)
        root = eng.new_seq()
        root.prefill(p, 64)
        history = [("prefill", p)]
        plain = eng.new_seq()
        leaves = [(root, history)]
        for i in range(5):
            s, h = leaves[i]
            own = A.stream_uniform(20 + i, "own", 3 + 4 * i, 0, 100)
            used = eng.new_seq()
            used.prefill(A.stream_uniform(40 + i, "used", 20, 0, 100), 64)
            used.decode(2, eng.num_layers)
            child = s.fork(into=used)
            child.prefill(own, 64)
            leaves.append((child, h + [("prefill", own)]))
        leaves[2][0].release()
        del leaves[2]
        st, toks = eng.decode_step([s for s, _ in leaves], eng.num_layers)
        assert st == 0
        for (s, h), t in zip(leaves, toks):
            plain.reset()
            for _, tokens in h:
                plain.prefill(tokens, 64)
            assert plain.decode(1, eng.num_layers) == [t] and plain.save() == s.save()
        for s, _ in leaves:
            s.reset()
    finally:
        eng.close()


@pytest.mark.parametrize("mode", [0, 2])
def test_attended_together_and_apart(gpu_lib, mode):
    """forks share pages: with mode 2 the rows of a step are attended together, with the same tokens"""
    set_mode, launches = gpu_lib.dll.sslm_b200_set_prefix_attention, gpu_lib.dll.sslm_b200_prefix_attention_launches
    launches.restype = C.c_uint64
    eng = engine(gpu_lib, "small", 128, 8)
    try:
        p = A.stream_uniform(3, "prompt", 50, 0, 100)
        root = eng.new_seq()
        root.prefill(p, 64)
        family = [root] + [root.fork() for _ in range(3)]
        # a second family, of the same sequence after a reset: other pages
        q = A.stream_uniform(4, "other", 37, 0, 100)
        root.reset()
        root.prefill(q, 64)
        family += [root.fork() for _ in range(2)]
        for i, s in enumerate(family):
            s.prefill(A.stream_uniform(50 + i, "own", 2 + i, 0, 100), 64)
        before = launches()
        assert set_mode(mode) == 0
        got = []
        for _ in range(4):
            st, toks = eng.decode_step(family, eng.num_layers)
            assert st == 0
            got.append(toks)
        assert (launches() > before) == (mode == 2)
        plain = eng.new_seq()
        for i in range(len(family)):
            plain.reset()
            plain.prefill(p if 1 <= i <= 3 else q, 64)
            plain.prefill(A.stream_uniform(50 + i, "own", 2 + i, 0, 100), 64)
            assert plain.decode(4, eng.num_layers) == [t[i] for t in got], i
    finally:
        set_mode(1)
        eng.close()


def test_adapters_schemas_and_history_go_along(gpu_lib):
    sh = A.SHAPES["small"]
    table = A.synthetic_schemas(0xF0, sh.vocab, 1)
    art = A.build_synthetic_model("small", 0xF0, 128, schemas=1)
    eng = abi.Engine(gpu_lib, art, blocks=4, max_batch=4, max_chunk=64)
    try:
        adapter = eng.map_adapter(A.build_synthetic_adapter(art, 5))
        h = C.c_void_p()
        assert gpu_lib.sslm_schema_lookup(eng.model, table[0]["name"].encode(), C.byref(h)) == 0
        p = A.stream_uniform(1, "prompt", 19, 0, sh.vocab - 1)
        settings = dict(repetition=60000, presence=9000, count_given=True)
        parent, plain = eng.new_seq(), eng.new_seq()
        for s in (parent, plain):
            assert gpu_lib.sslm_seq_set_schema(s.handle, h) == 0
            s.set_adapter(adapter)
            s.prefill(p, 64)
        plain.set_controls(**settings)
        a, b = parent.decode(1, eng.num_layers), None
        child = parent.fork()
        child.set_controls(**settings)                 # counts what the parent was given and made
        plain.set_controls(repetition=None)
        b = plain.decode(1, eng.num_layers)
        plain.set_controls(**settings)
        assert a == b
        for _ in range(3):
            st, toks = eng.decode_step([child, plain], eng.num_layers)
            assert st == 0 and toks[0] == toks[1]
            if toks[0] < 0:
                break
        assert child.save() == plain.save()
    finally:
        eng.close()


def test_a_pool_full_of_forks(gpu_lib):
    """every block credit used, every sequence to the end of its context"""
    eng = engine(gpu_lib, "tiny", 48, 6)
    try:
        root = eng.new_seq()
        root.prefill(A.stream_uniform(2, "prompt", 17, 0, 100), 64)
        seqs = [root] + [root.fork() for _ in range(5)]
        for i, s in enumerate(seqs):
            s.set_sampling(temperature=4.0, seed=i)
        n = 0
        while True:
            st, toks = eng.decode_step(seqs, eng.num_layers)
            if st != 0:
                break
            n += 1
        assert st == abi.ST["SSLM_CONTEXT_CAP_EXCEEDED"] and n == 48 - 17 + 1
        for _ in range(3):                              # and again, from sequences that are full
            for s in seqs[1:]:
                seqs[0].fork(into=s)
            assert all(s.save() == seqs[0].save() for s in seqs)
    finally:
        eng.close()


def test_refusals(gpu_lib):
    eng, other = engine(gpu_lib, "tiny", 48, 3), engine(gpu_lib, "tiny", 48, 2)
    fork = gpu_lib.dll.sslm_b200_seq_fork
    fork.restype, fork.argtypes = C.c_int, [C.c_void_p, C.c_void_p]
    bad, mid = abi.ST["SSLM_INVALID_ARGUMENT"], abi.ST["SSLM_SEQ_RESET_MIDTOKEN_REJECTED"]
    try:
        a, b, c = eng.new_seq(), eng.new_seq(), other.new_seq()
        for s in (a, b, c):
            s.prefill([1, 2, 3], 64)
        assert fork(None, a.handle) == bad and fork(a.handle, None) == bad and fork(a.handle, a.handle) == bad and fork(c.handle, a.handle) == bad
        a.decode(1, eng.num_layers)
        st, toks = eng.decode_step([a], 1)
        assert st == 0 and toks[0] == -1
        before = b.save()
        assert fork(b.handle, a.handle) == mid and fork(a.handle, b.handle) == mid
        assert b.save() == before
        a.decode(1, eng.num_layers)
        assert fork(b.handle, a.handle) == 0 and b.save() == a.save()
    finally:
        eng.close()
        other.close()
