"""sslm_b200_fork_resident and sslm_b200_compact_resident: page tables, holders and copies, against their definitions."""
import numpy as np
import pytest

from superslm_b200 import abi
from tests.support.resident_more import cache_case, compacted, forked

pytestmark = pytest.mark.gpu
OLD = -9


@pytest.fixture()
def torch():
    t = pytest.importorskip("torch")
    assert t.cuda.is_available()
    t.cuda.set_device(0)
    return t


class Fork:
    def __init__(self, lib, torch, case, parents, grow=None, copies=True):
        self.torch, self.case = torch, case
        self.parents = np.asarray(parents, dtype=np.int32)
        self.grow = None if grow is None else np.broadcast_to(np.asarray(grow, dtype=np.int32), self.parents.shape).copy()
        self.d = {k: torch.from_numpy(v).cuda() for k, v in case.items()}
        n, N = len(self.parents), len(case["holders"])
        full = lambda *shape: torch.full(shape, OLD, dtype=torch.int32, device="cuda")      # noqa: E731
        self.out = dict(out_holders=full(N), out_tables=full(*case["tables"].shape), out_lengths=full(n), drawn=full(N), moves=full(n, 2), counts=full(2), status=full(n))
        self.inputs = dict(parents=torch.from_numpy(self.parents).cuda(), grow=None if grow is None else torch.from_numpy(self.grow).cuda())
        self.call = abi.Fork(lib, self.d["kv"] if copies else None, self.d["holders"], self.d["tables"], self.d["lengths"], **self.inputs, **self.out)

    def check(self):
        self.call.run()
        self.torch.cuda.synchronize()
        return self.compare()

    def compare(self):
        grow = np.zeros_like(self.parents) if self.grow is None else self.grow
        want = forked(self.case, self.parents, grow, np.full_like(self.case["tables"], OLD))
        got = {k: v.cpu().numpy() for k, v in self.out.items()}
        for k in ("status", "out_lengths", "out_tables", "out_holders"):
            assert (got[k] == want[k]).all(), (k, np.argwhere(got[k] != want[k])[:5])
        m, n = len(want["moves"]), len(want["drawn"])
        assert got["counts"].tolist() == [m, n]
        assert (got["moves"][:m] == want["moves"]).all() and (got["moves"][m:] == OLD).all() and (got["drawn"][:n] == want["drawn"]).all()
        assert (self.d["kv"].cpu().numpy() == (want["kv"] if self.call.args.kv else self.case["kv"])).all()
        return want


def parents_of(seed, n, share=0.6, ended=0.1):
    g = np.random.default_rng(seed)
    p = np.where(g.random(n) < share, g.integers(0, n, n), np.arange(n))
    p[g.random(n) < ended] = -1
    return p


@pytest.mark.parametrize("sequences,longest", [(1, 0), (1, 16), (1, 17), (2, 40), (5, 15), (16, 100), (17, 300), (60, 33), (300, 500), (1000, 64), (3, 1500)])
@pytest.mark.parametrize("grow", [None, 1, 16, 50])
def test_forks(gpu_lib, torch, sequences, longest, grow):
    case = cache_case(1, sequences, longest, grow=grow or 0, spare=sequences * (2 + (grow or 0) // 16) + 9)
    Fork(gpu_lib, torch, case, parents_of(2, sequences), grow).check()


def test_all_from_one_and_all_ended(gpu_lib, torch):
    case = cache_case(3, 40, 200, spare=60)
    case["lengths"][7] = 199 if case["lengths"][7] == 0 else case["lengths"][7]
    case = cache_case(3, 40, 200, spare=60)
    f = Fork(gpu_lib, torch, case, np.full(40, 7))
    f.check()
    f = Fork(gpu_lib, torch, case, np.full(40, -1))
    want = f.check()
    assert (want["out_holders"] == 0).all()
    Fork(gpu_lib, torch, case, np.arange(40)).check()
    Fork(gpu_lib, torch, case, np.roll(np.arange(40), 1)).check()      # everyone becomes its neighbour: read as they were


@pytest.mark.parametrize("page_bytes,planes", [(16, 1), (512, 4), (1024, 7), (2048, 3), (2064, 2), (8192, 1)])
def test_pages_of_any_size(gpu_lib, torch, page_bytes, planes):
    case = cache_case(4, 21, 100, planes=planes, page_bytes=page_bytes, spare=60)
    Fork(gpu_lib, torch, case, parents_of(5, 21), 3 if case["tables"].shape[1] * 16 >= 103 else 0).check()


@pytest.mark.parametrize("free", [0, 1, 7, 30])
def test_too_few_pages(gpu_lib, torch, free):
    """those in front are served, the others stay what they were"""
    case = cache_case(6, 50, 90, shared=False, grow=20, spare=0)
    empty = np.flatnonzero(case["holders"] == 0)
    case["holders"][empty[free:]] = 1                          # (held by someone else)
    want = Fork(gpu_lib, torch, case, parents_of(7, 50), 20).check()
    assert (want["status"] == 102).any() and len(want["drawn"]) <= free


def test_refused_sequences_leave_the_others(gpu_lib, torch):
    case = cache_case(8, 20, 200, shared=False, spare=60)
    width = case["tables"].shape[1]
    case["lengths"][[3, 4, 5, 6, 9]] = -1, width * 16 + 1, 70, 90, 50
    case["tables"][5, 2] = -1
    case["tables"][6, 1] = len(case["holders"])
    parents = np.arange(20)
    parents[10:18] = 3, 4, 5, 6, -2, 20, 3, 9
    grow = np.zeros(20, dtype=np.int32)
    grow[0], grow[1], grow[9] = -1, width * 16, (1 << 31) - 1
    want = Fork(gpu_lib, torch, case, parents, grow).check()
    assert want["status"].tolist() == [7, 7, 0, 7, 7, 0, 0, 0, 0, 7, 7, 7, 101, 101, 101, 101, 7, 0, 0, 0]


def test_bad_pages_of_a_sequence_that_lets_go(gpu_lib, torch):
    """ids that do not exist are nobody's to let go"""
    case = cache_case(9, 6, 100, shared=False, spare=20)
    case["lengths"][2] = 40
    case["tables"][2, :3] = -5, 1 << 30, len(case["holders"])
    Fork(gpu_lib, torch, case, [0, 1, -1, 3, 4, 5]).check()
    Fork(gpu_lib, torch, case, [0, 1, 0, 3, 4, 5]).check()


def test_tables_alone_strided(gpu_lib, torch):
    case = cache_case(10, 12, 150, spare=40)
    f = Fork(gpu_lib, torch, case, parents_of(11, 12), copies=False)
    f.check()
    n, width = case["tables"].shape
    wide, out = torch.full((n, width + 5), -3, dtype=torch.int32, device="cuda"), torch.full((n, width + 9), OLD, dtype=torch.int32, device="cuda")
    wide[:, 3:3 + width] = f.d["tables"]
    f.call = abi.Fork(gpu_lib, None, f.d["holders"], wide[:, 3:3 + width], f.d["lengths"], **f.inputs, **dict(f.out, out_tables=out[:, 1:1 + width]))
    f.call.run()
    torch.cuda.synchronize()
    f.out["out_tables"].copy_(out[:, 1:1 + width])
    f.compare()
    assert (out[:, :1] == OLD).all() and (out[:, 1 + width:] == OLD).all()


def test_many_sequences(gpu_lib, torch):
    """the most there may be, a page table of one entry each"""
    n = 65535
    case = dict(kv=np.zeros((1, n + 900, 16), dtype=np.int8), holders=np.concatenate([np.ones(n), np.zeros(900)]).astype(np.int32),
                tables=np.arange(n, dtype=np.int32)[:, None], lengths=np.full(n, 5, dtype=np.int32))
    case["kv"][0, :, 0] = np.arange(n + 900) % 127
    parents = np.arange(n)
    parents[::73] = 65534
    Fork(gpu_lib, torch, case, parents, 1).check()


def test_fork_captured_and_replayed_with_compact(gpu_lib, torch):
    """steps of a search: fork, compact, fork again from what is left, captured once"""
    case = cache_case(12, 16, 120, grow=64, spare=200)
    f = Fork(gpu_lib, torch, case, parents_of(13, 16), 1)
    f.check()
    c = Compact(gpu_lib, torch, case)
    c.check()
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    d = {k: torch.from_numpy(v).cuda() for k, v in case.items()}
    full = lambda *shape: torch.full(shape, OLD, dtype=torch.int32, device="cuda")      # noqa: E731
    n, N = 16, len(case["holders"])
    f.call = abi.Fork(gpu_lib, d["kv"], d["holders"], d["tables"], d["lengths"], **f.inputs, **f.out)
    new_of, moves, counts = full(N), full(N // 2, 2), full(2)
    back = abi.Compact(gpu_lib, d["kv"], f.out["out_holders"], f.out["out_tables"], f.out["out_lengths"], out_holders=d["holders"], out_tables=d["tables"], new_of=new_of,
                       moves=moves, counts=counts)
    with torch.cuda.stream(stream):
        with torch.cuda.graph(graph, stream=stream):
            f.call.run()
            back.run()
            d["lengths"].copy_(f.out["out_lengths"])
    state = {k: v.copy() for k, v in case.items()}
    for step in range(4):
        parents = parents_of(20 + step, n, ended=0.0)
        f.inputs["parents"].copy_(torch.from_numpy(parents.astype(np.int32)))
        graph.replay()
        torch.cuda.synchronize()
        w = forked(state, parents, np.ones(n, dtype=np.int32), np.full_like(state["tables"], OLD))
        assert (w["status"] == 0).all()
        v = compacted(dict(kv=w["kv"], holders=w["out_holders"], tables=w["out_tables"], lengths=w["out_lengths"]), state["tables"])
        state = dict(kv=v["kv"], holders=v["out_holders"], tables=v["out_tables"], lengths=w["out_lengths"])
        for k in ("lengths", "holders", "kv"):
            assert (d[k].cpu().numpy() == state[k]).all(), (step, k)
        for i in range(n):
            used = -(-int(state["lengths"][i]) // 16)
            assert (d["tables"][i, :used].cpu().numpy() == state["tables"][i, :used]).all(), (step, i)


class Compact:
    def __init__(self, lib, torch, case, in_place=False, copies=True):
        self.torch, self.case, self.in_place = torch, case, in_place
        self.d = {k: torch.from_numpy(v).cuda() for k, v in case.items()}
        n, N = len(case["lengths"]), len(case["holders"])
        full = lambda *shape: torch.full(shape, OLD, dtype=torch.int32, device="cuda")      # noqa: E731
        self.out = dict(out_holders=full(N), out_tables=self.d["tables"] if in_place else full(*case["tables"].shape), new_of=full(N), moves=full(N // 2, 2), counts=full(2), status=full(n))
        self.call = abi.Compact(lib, self.d["kv"] if copies else None, self.d["holders"], self.d["tables"], self.d["lengths"], **self.out)

    def check(self):
        self.call.run()
        self.torch.cuda.synchronize()
        want = compacted(self.case, self.case["tables"] if self.in_place else np.full_like(self.case["tables"], OLD))
        got = {k: v.cpu().numpy() for k, v in self.out.items()}
        for k in ("status", "new_of", "out_tables", "out_holders"):
            assert (got[k] == want[k]).all(), (k, np.argwhere(got[k] != want[k])[:5])
        m = len(want["moves"])
        assert got["counts"].tolist() == [m, want["live"]] and (got["moves"][:m] == want["moves"]).all() and (got["moves"][m:] == OLD).all()
        kv = self.d["kv"].cpu().numpy()
        assert (kv == (want["kv"] if self.call.args.kv else self.case["kv"])).all()
        return want


@pytest.mark.parametrize("sequences,longest,spare", [(1, 0, 0), (1, 1, 0), (1, 16, 1), (2, 40, 100), (7, 200, 3), (40, 300, 500), (300, 200, 4000), (30, 100, 40000), (3, 1500, 50), (20, 700, 9000)])
@pytest.mark.parametrize("in_place", [False, True])
def test_compacts(gpu_lib, torch, sequences, longest, spare, in_place):
    Compact(gpu_lib, torch, cache_case(14, sequences, longest, spare=spare), in_place).check()


def test_nothing_free_and_nothing_used(gpu_lib, torch):
    case = cache_case(15, 9, 100)
    full = dict(case, holders=np.ones_like(case["holders"]))
    assert len(Compact(gpu_lib, torch, full).check()["moves"]) == 0
    empty = dict(case, holders=np.zeros_like(case["holders"]), lengths=np.zeros_like(case["lengths"]))
    assert Compact(gpu_lib, torch, empty).check()["live"] == 0
    half = dict(case, holders=(np.arange(len(case["holders"])) >= len(case["holders"]) // 2).astype(np.int32) * 5, lengths=np.zeros_like(case["lengths"]))
    Compact(gpu_lib, torch, half).check()


def test_bad_tables_leave_the_others(gpu_lib, torch):
    case = cache_case(16, 8, 200, shared=False, spare=90)
    case["lengths"][[1, 2, 3, 4, 5]] = -1, case["tables"].shape[1] * 16 + 1, 60, 60, 60
    case["tables"][3, 2] = -1
    case["tables"][4, 0] = len(case["holders"])
    case["tables"][5, 1] = np.flatnonzero(case["holders"] == 0)[0]
    want = Compact(gpu_lib, torch, case, copies=False).check()
    assert want["status"][:6].tolist() == [0, 7, 7, 101, 101, 101]


def test_planes_beyond_32_bits(gpu_lib, torch):
    """planes 2.6 GB apart"""
    case = cache_case(17, 6, 100, planes=2, page_bytes=2048, spare=30)
    f = Fork(gpu_lib, torch, case, parents_of(18, 6))
    N, used = 1_300_000, len(case["holders"])
    kv = torch.zeros((2, N, 2048), dtype=torch.int8, device="cuda")
    kv[:, N - used:] = f.d["kv"]
    holders = torch.ones(N, dtype=torch.int32, device="cuda")
    holders[N - used:] = f.d["holders"]
    out_holders, drawn = torch.zeros(N, dtype=torch.int32, device="cuda"), torch.zeros(N, dtype=torch.int32, device="cuda")
    abi.Fork(gpu_lib, kv, holders, f.d["tables"] + (N - used), f.d["lengths"], **f.inputs, **dict(f.out, out_holders=out_holders, drawn=drawn)).run()
    torch.cuda.synchronize()
    f.d["kv"].copy_(kv[:, N - used:])
    f.out["out_holders"].copy_(out_holders[N - used:])
    f.out["drawn"].copy_(drawn[:used] - (N - used))
    m = int(f.out["counts"][0])
    f.out["moves"][:m] -= N - used
    for i in range(6):
        k = -(-int(f.out["out_lengths"][i]) // 16)
        f.out["out_tables"][i, :k] -= N - used
    f.compare()
