"""Which rows are attended together when forks share pages on more than one level: behind an adopted prefix, behind forks of forks."""
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


class Family:
    """Sequences of one engine with what each was given, and a sequence by itself that is given the same."""

    def __init__(self, lib, cap, blocks, shape="tiny"):
        sh = A.SHAPES[shape]
        self.vocab = sh.vocab
        self.eng = abi.Engine(lib, A.build_synthetic_model(shape, 0xF1, cap), blocks=blocks + 1, max_batch=blocks, max_chunk=512)
        self.given = {}

    def tokens(self, name, n):
        return A.stream_uniform(n, name, n, 0, self.vocab - 1).tolist()

    def more(self, s, name, n):
        t = self.tokens(name, n)
        s.prefill(t, 512)
        self.given[s] = self.given.get(s, []) + t
        return s

    def new(self, name, n):
        return self.more(self.eng.new_seq(), name, n)

    def adopted(self, n, times):
        lib, h, t = self.eng.lib, C.c_void_p(), np.asarray(self.tokens("prefix", n), dtype=np.int32)
        assert lib.sslm_prefix_begin(self.eng.model, C.byref(self.eng.pool), C.byref(h)) == 0
        c = C.c_int32(0)
        for at in range(0, n, 512):
            part = t[at:at + 512]
            assert lib.sslm_prefix_prefill(self.eng.model, h, part.ctypes.data_as(C.POINTER(C.c_int32)), len(part), 512, 0, self.eng.ws, C.byref(c)) == 0 and c.value == len(part)
        assert lib.sslm_prefix_freeze(h) == 0
        out = []
        for _ in range(times):
            s = self.eng.new_seq()
            assert lib.sslm_seq_adopt_prefix(s.handle, h) == 0
            self.given[s] = t.tolist()
            out.append(s)
        assert lib.sslm_prefix_release(h) == 0
        return out

    def fork(self, s):
        child = s.fork()
        self.given[child] = list(self.given[s])
        return child

    def check(self, dll, mode, steps=3, plain=True):
        """launches of the kernel that attends rows together; the tokens are those of the sequences by themselves"""
        seqs = list(self.given)
        assert dll.sslm_b200_set_prefix_attention(mode) == 0
        before, got = dll.sslm_b200_prefix_attention_launches(), []
        for _ in range(steps):
            st, toks = self.eng.decode_step(seqs, self.eng.num_layers)
            assert st == 0
            got.append(toks)
        launches = dll.sslm_b200_prefix_attention_launches() - before
        if plain:
            alone = self.eng.new_seq()
            for i, s in enumerate(seqs):
                alone.reset()
                alone.prefill(self.given[s], 512)
                assert alone.decode(steps, self.eng.num_layers) == [t[i] for t in got], i
                assert alone.save() == s.save()
        return launches


@pytest.mark.parametrize("prefix", [9, 16])
def test_forks_behind_an_adopted_prefix_of_a_page_or_less(gpu_lib, dll, prefix):
    """their own pages are what they share"""
    f = Family(gpu_lib, 128, 5)
    try:
        root = f.more(f.adopted(prefix, 1)[0], "own", 60)
        for _ in range(4):
            f.fork(root)
        assert f.check(dll, 2) > 0
    finally:
        f.eng.close()


# 8 rows behind 4,096 positions and more are attended together by themselves (8 x 4,112^2 is above 2^27); behind a page or two they are not
LONG = 4112


@pytest.mark.parametrize("first", ["adopted", "forked"])
def test_forks_share_what_their_parent_has_by_then(gpu_lib, dll, first):
    f = Family(gpu_lib, LONG + 128, 9)
    try:
        if first == "adopted":
            root = f.adopted(32, 1)[0]
        else:
            root = f.new("start", 33)
            other = f.fork(root)
            del f.given[other]
        f.more(root, "own", LONG)
        for _ in range(7):
            f.fork(root)
        assert f.check(dll, 1, steps=2) > 0
    finally:
        f.eng.close()


def test_a_fork_takes_nothing_from_the_prefix_that_many_share(gpu_lib, dll):
    """8 rows behind one long prefix, two of which share a page more, are attended behind the prefix as before"""
    f = Family(gpu_lib, LONG + 128, 8)
    try:
        seqs = f.adopted(LONG, 7)
        for i, s in enumerate(seqs):
            f.more(s, "own%d" % i, 17 + i)
        f.fork(seqs[3])
        assert f.check(dll, 1, steps=2) > 0
    finally:
        f.eng.close()


@pytest.mark.parametrize("mode", [0, 2])
def test_families_inside_families(gpu_lib, dll, mode):
    """forks of forks of adopters, of many levels, parents that go on and that end, and sequences beside them"""
    f = Family(gpu_lib, 256, 22, "small")
    try:
        a, b, c = f.adopted(40, 3)
        f.more(b, "b", 3)
        f.new("beside", 21)
        front = [a]
        for level in range(7):                     # deeper by more than a page each time
            s = f.fork(front[-1])
            f.more(front[-1], "left%d" % level, 1 + level)
            f.more(s, "down%d" % level, 18 + level)
            front.append(s)
        for s in front[2:5]:
            f.more(f.fork(s), "twig", 2)
        f.more(f.fork(f.more(c, "c", 30)), "d", 1)
        gone = front[3]
        del f.given[gone]
        gone.release()
        again = f.fork(front[6])
        f.more(again, "e", 20)
        f.more(f.fork(again), "f", 20)
        assert (f.check(dll, mode) > 0) == (mode == 2)
    finally:
        f.eng.close()
