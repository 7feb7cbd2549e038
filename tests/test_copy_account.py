"""The account of a block's bulk copies (csrc/sslm_copies.h), compiled for the host and led through a model of the barriers: whatever wait runs
out, no copy is asked for into a place whose last one is still open, and the block waits for every place's last copy, by the turn that it is in."""
import ctypes as C
import os
import random
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SOURCE = """
#include "superslm_b200/csrc/sslm_copies.h"
using sslm::CopyAccount;
extern "C" {
uint32_t acc_place(const CopyAccount* a, uint32_t c) { return a->place(c); }
uint32_t acc_parity(const CopyAccount* a, uint32_t c) { return a->parity(c); }
uint32_t acc_begin(CopyAccount* a, uint32_t before, uint32_t chunks) { return a->begin(before, chunks); }
int acc_follows(CopyAccount* a, uint32_t i, uint32_t chunks, int late) { return a->follows(i, chunks, late != 0); }
uint32_t acc_open(const CopyAccount* a) { return a->open(); }
}
"""


class Account(C.Structure):
    _fields_ = [("places", C.c_uint32), ("issued", C.c_uint32)]


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    d = tmp_path_factory.mktemp("copies")
    (d / "shim.cpp").write_text(SOURCE)
    subprocess.run(["g++", "-O1", "-std=c++17", "-fPIC", "-shared", "-I", ROOT, "-o", str(d / "shim.so"), str(d / "shim.cpp")], check=True)
    return C.CDLL(str(d / "shim.so"))


def block(lib, places, passes, late_at):
    """One block over passes of so many chunks each, the wait for chunk `late_at` running out (None: no wait does). Returns the chunks
    asked for, and (chunk, parity) of the waits at the end."""
    a = Account(places, 0)
    at = C.byref(a)
    asked, last = [], {}      # last: a place's newest chunk

    def issue(chunk):
        p = lib.acc_place(at, chunk)
        if p in last:
            assert last[p] in used and last[p] != late_at, "a place whose last copy is open"
            assert lib.acc_parity(at, last[p]) != lib.acc_parity(at, chunk)
        last[p] = chunk
        asked.append(chunk)
    used, before, late = set(), 0, False
    for chunks in passes:
        if late:
            break
        for i in range(lib.acc_begin(at, before, chunks)):
            issue(before + i)
        for i in range(chunks):
            if not late:
                assert last[lib.acc_place(at, before + i)] == before + i
                late = before + i == late_at
                if not late:
                    used.add(before + i)
            if lib.acc_follows(at, i, chunks, late):
                issue(before + i + places)
        before += chunks
    assert a.issued == len(asked) and asked == list(range(a.issued))
    waits = [(c, lib.acc_parity(at, c)) for c in range(lib.acc_open(at), a.issued)] if late else []
    return asked, waits, last, lib


@pytest.mark.parametrize("places", [1, 2, 3, 4])
def test_every_open_copy_is_waited_for(lib, places):
    r = random.Random(places)
    for _ in range(4000):
        passes = [r.randrange(0, 14) for _ in range(r.randrange(1, 5))]
        total = sum(passes)
        late_at = r.choice([None] + list(range(total)))
        asked, waits, last, _ = block(lib, places, passes, late_at)
        if late_at is None:
            assert len(asked) == total and waits == []
            continue
        assert sorted(c for c, _ in waits) == sorted(last.values())      # each place's last copy, whatever was used of them
        assert late_at in last.values()


def test_ten_chunks_in_four_places_late_at_the_first(lib):
    asked, waits, _, _ = block(lib, 4, [10], 0)
    assert asked == [0, 1, 2, 3] and waits == [(0, 0), (1, 0), (2, 0), (3, 0)]
