"""sslm_b200_attention_prefix_resident: integer attention of rows that share prefixes, against its definition in 64 bits. All
results are integers and have to be equal."""
import ctypes as C

import numpy as np
import pytest

from superslm_b200 import abi
from tests.support.resident import attention_case, attention_rows

pytestmark = pytest.mark.gpu

SHAPES = {"0.5b": (14, 2, 64), "1.5b": (12, 2, 128), "3b": (16, 2, 128), "tiny": (4, 2, 32), "mha": (3, 3, 64), "mqa": (5, 1, 32), "wide": (8, 8, 128),
          "g7": (7, 1, 128), "g1": (2, 2, 32), "g3": (6, 2, 64), "g1w": (2, 2, 128)}


@pytest.fixture()
def torch():
    t = pytest.importorskip("torch")
    assert t.cuda.is_available()
    t.cuda.set_device(0)
    return t


@pytest.fixture()
def splits(gpu_lib):
    f = gpu_lib.dll.sslm_b200_set_attention_splits
    yield lambda n: f(n)
    f(0)


JUNK = 0x5A5A5A5A


class Call:
    def __init__(self, lib, torch, case, extra_rows=0, **more):
        self.case, self.torch = case, torch
        self.d = {k: (None if v is None else torch.from_numpy(v).cuda()) for k, v in case.items()}
        rows, heads, hd = case["q"].shape
        self.out = torch.full((rows, heads, hd), JUNK, dtype=torch.int32, device="cuda")
        self.status = torch.full((rows,), 77, dtype=torch.int32, device="cuda")
        self.call = abi.PrefixAttention(lib, out=self.out, row_status=self.status, **self.d, **more)

    def check(self, want=None, refused=()):
        self.call.run()
        self.torch.cuda.synchronize()
        self.compare(want, refused)

    def compare(self, want=None, refused=()):
        want = attention_rows(self.case) if want is None else want
        out, status = self.out.cpu().numpy(), self.status.cpu().numpy()
        for r in range(len(out)):
            if r in want and r not in refused:
                assert status[r] == 0, (r, status[r])
                assert (out[r] == want[r]).all(), (r, int((out[r] != want[r]).sum()), out[r].ravel()[:8], want[r].ravel()[:8])
            else:
                assert (out[r] == JUNK).all(), r
                assert status[r] == (refused[r] if r in refused else 77), (r, status[r])


def lengths(seed, n, lo, hi):
    return np.random.default_rng(seed).integers(lo, hi + 1, n)


@pytest.mark.parametrize("shape", sorted(SHAPES))
@pytest.mark.parametrize("rows,prefix,lo,hi", [(1, [0], 1, 1), (1, [1], 0, 0), (3, [16], 1, 17), (9, [300], 0, 40), (33, [129], 1, 3), (40, [127, 0, 513], 0, 70)])
def test_small_batches(gpu_lib, torch, shape, rows, prefix, lo, hi):
    Call(gpu_lib, torch, attention_case(rows + len(shape), SHAPES[shape], prefix, lengths(rows, rows, lo, hi))).check()


@pytest.mark.parametrize("n", [1, 2, 4, 8, 16])
@pytest.mark.parametrize("shape,rows,prefix,hi", [("1.5b", 21, [700], 100), ("0.5b", 7, [1000, 33], 60), ("tiny", 64, [260, 0, 5], 200), ("mqa", 2, [2000], 9),
                                                  ("g1", 30, [515], 130)])
def test_every_cut_gives_the_same(gpu_lib, torch, splits, n, shape, rows, prefix, hi):
    """one block a tile up to clusters of sixteen, tiles of sixteen and of thirty-two query rows"""
    case = attention_case(rows, SHAPES[shape], prefix, lengths(rows, rows, 0, hi))
    want = attention_rows(case)
    assert splits(n) == 0
    Call(gpu_lib, torch, case).check(want)


@pytest.mark.parametrize("shape,rows,prefix,lo,hi", [("1.5b", 64, [2048], 16, 256), ("0.5b", 100, [900, 17, 0, 333], 1, 300), ("3b", 5, [8000], 1, 100), ("tiny", 256, [640], 0, 30)])
def test_larger_batches(gpu_lib, torch, shape, rows, prefix, lo, hi):
    Call(gpu_lib, torch, attention_case(rows, SHAPES[shape], prefix, lengths(rows + 1, rows, lo, hi))).check()


@pytest.mark.parametrize("shape,prefix,suffix", [("3b", [32768], [0, 0, 0]), ("tiny", [32700], [68, 1]), ("1.5b", [0], [32768, 5]), ("mqa", [16385], [16383, 0, 7]),
                                                 ("g1", [0, 0], [32768] * 3), ("g1w", [0], [32768, 32000] + [31000] * 14), ("g1w", [16384], [16384] * 16),
                                                 ("g3", [30000], [2768] * 11), ("0.5b", [0], [32768] * 2)])
def test_widest_rows(gpu_lib, torch, shape, prefix, suffix):
    Call(gpu_lib, torch, attention_case(5, SHAPES[shape], prefix, suffix)).check()


@pytest.mark.parametrize("shape", sorted(SHAPES))
@pytest.mark.parametrize("prefix,suffix", [([300, 0], [40, 0, 7] + [100] * 30), ([20000], [12768, 12767] + [60] * 9)])
def test_both_maxima_at_their_limit(gpu_lib, torch, shape, prefix, suffix):
    """page tables that hold 32,768 positions each: tiles of fewer rows, whatever the shape"""
    Call(gpu_lib, torch, attention_case(6, SHAPES[shape], prefix, suffix, widths=(2048, 2048))).check()


def test_a_row_longer_than_the_longest(gpu_lib, torch):
    case = attention_case(7, SHAPES["tiny"], [32760], [8, 9, 0, 300, 1])
    Call(gpu_lib, torch, case).check(refused={1: 7, 3: 7})


@pytest.mark.parametrize("consts", [(1, 1, 0), (1, 11_863_283, 0), ((1 << 23), (1 << 23), 0), (5, 11, (1 << 40)), (3000, 6000, 0), (1 << 20, 1 << 21, 1 << 46),
                                    (11_863_283, 11_863_283, 0)])
@pytest.mark.parametrize("deviation", [0.0, 3.0, 400.0])
def test_constants_at_the_edges_of_their_domain(gpu_lib, torch, consts, deviation):
    """all scores equal, close together, and saturated codes (-128 among them); probabilities at their exact borders"""
    case = attention_case(int(deviation) + consts[0], SHAPES["1.5b"], [150], [3, 40, 0, 17, 1], deviation=deviation, consts=consts)
    Call(gpu_lib, torch, case).check()


def test_rows_that_see_nothing(gpu_lib, torch):
    case = attention_case(1, SHAPES["0.5b"], [0, 20, 0], [0, 5, 0, 0, 3, 0], per_group=[3, 1, 2])
    case["fold"] = None
    c = Call(gpu_lib, torch, case)
    c.check()
    assert (c.out[0] == 0).all() and (c.out[2] == 0).all() and (c.out[5] == 0).all()
    case = attention_case(2, SHAPES["1.5b"], [0], [0] * 9)
    Call(gpu_lib, torch, case, max_prefix=0, max_suffix=0).check()


def test_rows_outside_the_groups_are_left_alone(gpu_lib, torch):
    case = attention_case(3, SHAPES["1.5b"], [40, 9], lengths(3, 12, 1, 30), per_group=[4, 8])
    case["group_start"] = np.array([2, 5, 9], dtype=np.int32)
    Call(gpu_lib, torch, case).check()
    case["group_start"] = np.array([4, 4, 4], dtype=np.int32)
    Call(gpu_lib, torch, case).check(want={})


def test_more_groups_than_a_warp_looks_at_at_once(gpu_lib, torch):
    """groups of none, one and several rows, in tiles that lie behind 32, 64, ... groups"""
    g = np.random.default_rng(9)
    per = g.choice([0, 1, 2, 5, 11], 150)
    per[[0, 31, 32, 63, 64, 149]] = [0, 7, 0, 9, 1, 3]
    n = int(per.sum())
    case = attention_case(9, SHAPES["tiny"], g.integers(0, 40, 150).tolist(), lengths(9, n, 0, 20), per_group=per.tolist())
    Call(gpu_lib, torch, case).check()


@pytest.mark.parametrize("per_group", [65535, 1])
def test_as_many_rows_as_a_call_takes(gpu_lib, torch, per_group):
    """65,535 rows of one group, and as many groups of a row: copies of 13 rows"""
    n, one = 65535, attention_case(10, SHAPES["mqa"], [33], lengths(10, 13, 0, 40))
    want = attention_rows(one)
    at = np.arange(n) % 13
    case = dict(one, **{k: one[k][at] for k in ("q", "consts", "suffix_len", "suffix_pages")})
    if per_group == 1:
        case.update(group_start=np.arange(n + 1, dtype=np.int32), prefix_len=np.full(n, 33, dtype=np.int32), prefix_pages=np.repeat(one["prefix_pages"], n, 0))
    else:
        case["group_start"] = np.array([0, n], dtype=np.int32)
    c = Call(gpu_lib, torch, case)
    c.call.run()
    torch.cuda.synchronize()
    assert (c.status.cpu().numpy() == 0).all()
    assert (c.out.cpu().numpy() == np.stack([want[r] for r in range(13)])[at]).all()


def test_draft_tokens_share_their_suffix_pages(gpu_lib, torch):
    case = attention_case(4, SHAPES["0.5b"], [100], np.repeat([7, 16, 31, 1], 4) + np.tile(np.arange(4), 4))
    case["suffix_pages"] = np.repeat(case["suffix_pages"][::4], 4, axis=0).copy()
    Call(gpu_lib, torch, case).check()


@pytest.mark.parametrize("splits_n", [0, 4])
def test_refused_rows_leave_the_others(gpu_lib, torch, splits, splits_n):
    splits(splits_n)
    n = 14
    case = attention_case(6, SHAPES["1.5b"], [70, 50], lengths(6, n, 17, 60), per_group=[8, 6])
    good = attention_rows(case)
    pages = case["kv"].shape[2]
    case["suffix_pages"][1, 1] = pages
    case["suffix_pages"][2, 0] = -1
    case["suffix_len"][3] = -1
    case["suffix_len"][4] = 16 * case["suffix_pages"].shape[1] + 1
    case["consts"][5, 1, 0] = 0                                     # q_ln2 < 1
    case["consts"][6, 0, 0] = case["consts"][6, 0, 1] + 1           # q_ln2 > q_b
    case["consts"][7, 0, 2] = -1
    case["consts"][8, 1, 1] = 1 << 24
    case["consts"][9, 1, 2] = 1 << 47                               # peak
    case["consts"][10] = [1, 1, (1 << 47) - 1]                      # peak in range, 2^47 * width < 2^63: not refused
    refused = {1: 101, 2: 101, 3: 7, 4: 7, 5: 20, 6: 20, 7: 20, 8: 20, 9: 20}
    want = {r: v for r, v in good.items() if r not in refused}
    want.update(attention_rows(case, only={10}))
    Call(gpu_lib, torch, case).check(want, refused)


def test_a_bad_prefix_refuses_its_group_only(gpu_lib, torch):
    case = attention_case(7, SHAPES["0.5b"], [100, 90, 33], lengths(7, 30, 1, 20))
    good = attention_rows(case)
    case["prefix_pages"][1, 5] = 1 << 30
    Call(gpu_lib, torch, case).check(good, {r: 101 for r in range(10, 20)})
    case["prefix_pages"][1, 5] = 0
    case["prefix_len"][1] = -5
    Call(gpu_lib, torch, case).check(good, {r: 7 for r in range(10, 20)})
    case["prefix_len"][1] = 113      # (the table has room for 112)
    Call(gpu_lib, torch, case).check(good, {r: 7 for r in range(10, 20)})
    # a bad id behind the prefix's end is not read
    case["prefix_len"][1] = 16
    case["prefix_pages"][1, 1:] = -7
    Call(gpu_lib, torch, case).check()


def test_strided_rows(gpu_lib, torch):
    case = attention_case(8, SHAPES["1.5b"], [77], lengths(8, 11, 0, 33))
    c = Call(gpu_lib, torch, case)
    heads, hd = case["q"].shape[1:]
    wide_q = torch.zeros((11, heads * hd + 36), dtype=torch.int8, device="cuda")
    q = wide_q[:, 4:4 + heads * hd].view(11, heads, hd)
    q.copy_(c.d["q"])
    wide_out = torch.full((11, heads + 3, hd), JUNK, dtype=torch.int32, device="cuda")
    out = wide_out[:, 2:2 + heads]
    tables = torch.full((11, 40), -9, dtype=torch.int32, device="cuda")
    tables[:, 7:7 + c.d["suffix_pages"].shape[1]] = c.d["suffix_pages"]
    args = dict(c.d, q=q, suffix_pages=tables[:, 7:7 + c.d["suffix_pages"].shape[1]])
    abi.PrefixAttention(gpu_lib, out=out, row_status=c.status, **args).run()
    torch.cuda.synchronize()
    c.out.copy_(out)
    c.compare()
    assert (wide_out[:, :2] == JUNK).all() and (wide_out[:, 2 + heads:] == JUNK).all()


def test_offsets_beyond_32_bits(gpu_lib, torch):
    """a pool of 2.6 GB planes: pages of the second plane of the second kv head lie beyond 2^32 bytes"""
    case = attention_case(9, (12, 2, 128), [100], [20, 5, 33])
    small = case["kv"]
    pages, total = small.shape[2], 1_300_000
    where = np.sort(np.random.default_rng(1).choice(total, pages, replace=False))
    where[-1] = total - 1
    big = torch.empty((2, 2, total, 2048), dtype=torch.int8, device="cuda")
    big[:, :, torch.from_numpy(where).cuda()] = torch.from_numpy(small).cuda()
    moved = dict(case, prefix_pages=where[case["prefix_pages"]].astype(np.int32), suffix_pages=where[case["suffix_pages"]].astype(np.int32))
    want = attention_rows(case)
    c = Call(gpu_lib, torch, dict(moved, kv=small))
    abi.PrefixAttention(gpu_lib, out=c.out, row_status=c.status, **dict(c.d, kv=big)).run()
    torch.cuda.synchronize()
    c.compare(want)


def funnel(port, row, site):
    from oracle.harness import Scale
    codes, sc = np.zeros(row.size, dtype=np.int8), Scale()
    row = np.ascontiguousarray(row.ravel(), dtype=np.int64)
    st = port.osc_funnel(row.ctypes.data, row.size, None, 0, Scale(*site), codes.ctypes.data, C.byref(sc))
    return codes, (sc.m, sc.e), st


def test_codes_feed_the_linear_layer(gpu_lib, torch, port):
    """context codes and scales against the oracle's funnel, and the chain they are for: attention, then the output projection"""
    from tests.test_gpu_parity import oracle_linear
    case = attention_case(10, SHAPES["1.5b"], [500, 0], lengths(10, 20, 0, 50))
    case["fold"][:] = [1, 0, 0]
    case["consts"][4, 1, 0] = 0
    rows, width = 20, 1536
    site = (1090717716, -44)
    codes = torch.full((rows, width), 0x5A, dtype=torch.int8, device="cuda")
    scales = torch.full((rows, 2), -1, dtype=torch.int64, device="cuda")
    c = Call(gpu_lib, torch, case, site=site, out_codes=codes, out_scales=scales)
    g = np.random.default_rng(2)
    w = g.integers(-127, 128, (640, width)).astype(np.int8)
    fold = np.stack([np.zeros(640), g.integers(1 << 30, 1 << 31, 640), g.integers(8, 21, 640)], 1).astype(np.int32)
    dw, dfold = torch.from_numpy(w).cuda(), torch.from_numpy(fold).cuda()
    folded = torch.zeros((rows, 640), dtype=torch.int32, device="cuda")
    f = gpu_lib.dll.sslm_b200_linear_resident
    f.argtypes = [C.c_void_p] * 3 + [C.c_int32] * 3 + [C.c_void_p, C.c_int64, C.c_int64] + [C.c_void_p] * 5
    c.call.run()
    assert f(codes.data_ptr(), dw.data_ptr(), dfold.data_ptr(), rows, 640, width, scales.data_ptr(), *site, folded.data_ptr(), None, None, None, None) == 0
    torch.cuda.synchronize()
    want = attention_rows(case, only=set(range(rows)) - {4})
    c.compare(want, {4: 20})
    got, gots, gotf = codes.cpu().numpy(), scales.cpu().numpy(), folded.cpu().numpy()
    assert (got[4] == 0x5A).all() and (gots[4] == -1).all()
    keep = [r for r in range(rows) if r != 4]
    for r in keep:
        wc, ws, st = funnel(port, want[r], site)
        assert st == 0 and (got[r] == wc).all() and tuple(gots[r]) == ws, r
    full = oracle_linear(got[keep], w, fold, gots[keep], site)
    assert (gotf[keep] == full[0]).all()


def test_captured_and_replayed_with_other_lengths(gpu_lib, torch):
    cases = [attention_case(s, SHAPES["0.5b"], [200, 100], lengths(s, 16, 0, 60)) for s in (20, 21, 22)]
    room = max(c["suffix_pages"].shape[1] for c in cases)
    pool = max(c["kv"].shape[2] for c in cases)
    for c in cases:
        c["suffix_pages"] = np.pad(c["suffix_pages"], ((0, 0), (0, room - c["suffix_pages"].shape[1])))
        c["kv"] = np.pad(c["kv"], ((0, 0), (0, 0), (0, pool - c["kv"].shape[2]), (0, 0)))
    cases[1]["group_start"] = np.array([0, 3, 16], dtype=np.int32)
    cases[2]["prefix_len"] = np.array([0, 77], dtype=np.int32)
    c = Call(gpu_lib, torch, cases[0])
    c.check()
    stream = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream):
        with torch.cuda.graph(graph, stream=stream):
            c.call.run()
    for case in cases[1:] + cases[:1]:
        for k, v in case.items():
            c.d[k].copy_(torch.from_numpy(v))
        c.out.fill_(JUNK)
        c.status.fill_(77)
        c.case = case
        graph.replay()
        torch.cuda.synchronize()
        c.compare()


def test_calls_on_two_streams(gpu_lib, torch):
    calls = [Call(gpu_lib, torch, attention_case(30 + i, SHAPES["1.5b"], [600], lengths(30 + i, 24, 1, 50))) for i in range(2)]
    streams = [torch.cuda.Stream() for _ in calls]
    torch.cuda.synchronize()
    for _ in range(20):
        for c, s in zip(calls, streams):
            c.call.run(s.cuda_stream)
    torch.cuda.synchronize()
    for c in calls:
        c.compare()


@pytest.mark.parametrize("splits_n,exchange", [(4, 0), (4, 1), (4, 2), (4, 3), (1, 3)])
def test_a_wait_that_runs_out(gpu_lib, torch, splits, splits_n, exchange):
    """block 0 waits for more than its peers send, or its copies of V bring: its rows are reported, the next call is right"""
    arm = gpu_lib.dll.sslm_b200_debug_withhold_exchange
    arm.argtypes = [C.c_int32, C.c_int32]
    assert arm(6, 4) == abi.ST["SSLM_INVALID_ARGUMENT"]
    splits(splits_n)
    c = Call(gpu_lib, torch, attention_case(40, SHAPES["1.5b"], [600], lengths(40, 5, 1, 50)))
    try:
        assert arm(6, exchange) == 0
        c.call.run()
        torch.cuda.synchronize()
    finally:
        arm(-1, 0)
    # (exchanges of a cluster of four: two rows a tile, or five)
    assert c.status[0] == 100 and all(s in (0, 100) for s in c.status.tolist())
    c.out.fill_(JUNK)
    c.check()


def test_empty_calls(gpu_lib, torch):
    case = attention_case(50, SHAPES["tiny"], [5], [1, 2])
    c = Call(gpu_lib, torch, case)
    c.call.args.rows = 0
    c.check(want={})
    c.call.args.rows, c.call.args.groups = 2, 0
    c.check(want={})


@pytest.mark.parametrize("shape", ["1.5b", "g7", "0.5b", "tiny"])
@pytest.mark.parametrize("splits_n", [1, 4])
def test_a_pool_at_any_16_byte_boundary(gpu_lib, torch, splits, splits_n, shape):
    splits(splits_n)
    case = attention_case(60, SHAPES[shape], [130, 33], lengths(60, 9, 0, 50))
    want = attention_rows(case)
    c = Call(gpu_lib, torch, case)
    raw = torch.zeros(c.d["kv"].numel() + 64, dtype=torch.int8, device="cuda")
    for first in (16, 48, 32):
        kv = raw[first:first + c.d["kv"].numel()].view(c.d["kv"].shape)
        kv.copy_(c.d["kv"])
        assert kv.data_ptr() % 32 == first % 32
        c.out.fill_(JUNK)
        c.status.fill_(77)
        abi.PrefixAttention(gpu_lib, out=c.out, row_status=c.status, **dict(c.d, kv=kv)).run()
        torch.cuda.synchronize()
        c.compare(want)
