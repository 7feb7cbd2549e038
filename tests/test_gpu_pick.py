"""sslm_b200_pick_resident: penalties, biases and masks on logits and the greedy token, against the definition in 64 bits."""
import ctypes as C

import numpy as np
import pytest

from superslm_b200 import abi
from tests.support.resident import LOWEST, changed_logits, picked

pytestmark = pytest.mark.gpu


@pytest.fixture()
def torch():
    t = pytest.importorskip("torch")
    assert t.cuda.is_available()
    t.cuda.set_device(0)
    return t


def make(seed, rows, vocab, history=0, bias=0, masks=None, spread=60000, params=True):
    g = np.random.default_rng(seed)
    c = dict(logits=np.rint(g.normal(0, spread, (rows, vocab))).astype(np.int32), params=None, history=None, history_len=None, bias_tokens=None, bias_values=None,
             bias_len=None, masks=None, mask_page=None)
    if params:
        c["params"] = np.stack([g.integers(20000, 60000, rows), g.integers(-30000, 60000, rows), g.integers(-3000, 9000, rows)], 1).astype(np.int32)
    if history:
        c["history"] = (g.random((rows, history)) ** 3 * vocab * 1.02 - 0.01 * vocab).astype(np.int32)      # (some ids outside the vocabulary)
        c["history_len"] = g.integers(0, history + 1, rows).astype(np.int32)
        c["history_len"][0] = history
    if bias:
        c["bias_tokens"] = g.integers(-2, vocab + 2, (rows, bias)).astype(np.int32)
        c["bias_tokens"][:, :bias // 2] = c["bias_tokens"][:, bias - bias // 2:]                            # (the same token twice)
        c["bias_values"] = g.integers(-400000, 400000, (rows, bias)).astype(np.int32)
        c["bias_len"] = g.integers(0, bias + 1, rows).astype(np.int32)
        c["bias_len"][0] = bias
    if masks is not None:
        bits = g.random((5, (vocab + 7) // 8 * 8)) < masks
        bits[4] = False
        c["masks"] = np.packbits(bits, axis=1, bitorder="little")
        c["mask_page"] = g.integers(-1, 5, rows).astype(np.int32)
        c["mask_page"][-1] = 4
    return c


def row_of(c, r):
    n = 0 if c["history"] is None else c["history_len"][r]
    m = 0 if c["bias_tokens"] is None else c["bias_len"][r]
    return changed_logits(c["logits"][r], None if c["params"] is None else c["params"][r], () if n == 0 else c["history"][r, :n],
                          () if m == 0 else list(zip(c["bias_tokens"][r, :m].tolist(), c["bias_values"][r, :m].tolist())),
                          None if c["masks"] is None or c["mask_page"][r] < 0 else c["masks"][c["mask_page"][r]])


class Call:
    def __init__(self, lib, torch, case, logits=True, **more):
        self.torch, self.case = torch, case
        self.d = {k: None if v is None else torch.from_numpy(v).cuda() for k, v in case.items()}
        rows = case["logits"].shape[0]
        self.tokens = torch.full((rows,), 55, dtype=torch.int32, device="cuda")
        self.best = torch.full((rows,), 55, dtype=torch.int32, device="cuda")
        self.status = torch.full((rows,), 77, dtype=torch.int32, device="cuda")
        self.out = torch.full(case["logits"].shape, 55, dtype=torch.int32, device="cuda") if logits else None
        self.call = abi.Pick(lib, out_tokens=self.tokens, out_best=self.best, out_logits=self.out, row_status=self.status, **dict(self.d, **more))

    def check(self, refused=()):
        self.call.run()
        self.torch.cuda.synchronize()
        self.compare(refused)

    def compare(self, refused=()):
        tokens, best, status = self.tokens.cpu().numpy(), self.best.cpu().numpy(), self.status.cpu().numpy()
        out = None if self.out is None else self.out.cpu().numpy()
        for r in range(len(tokens)):
            if r in refused:
                assert status[r] == refused[r] and tokens[r] == best[r] == 55 and (out is None or (out[r] == 55).all()), r
                continue
            want = row_of(self.case, r)
            assert status[r] == 0
            if out is not None:
                assert (out[r] == want).all(), (r, np.flatnonzero(out[r] != want)[:5], out[r][out[r] != want][:5], want[out[r] != want][:5])
            assert (tokens[r], best[r]) == picked(want), r


@pytest.mark.parametrize("vocab", [1, 2, 3, 5, 31, 32, 33, 127, 512, 4097, 8191, 8193, 32003, 151936])
@pytest.mark.parametrize("rows,history,bias,masks", [(1, 0, 0, None), (3, 40, 5, 0.5), (6, 700, 0, None), (2, 0, 33, 0.02), (5, 9, 1, 0.9)])
def test_rows(gpu_lib, torch, vocab, rows, history, bias, masks):
    case = make(vocab + rows, rows, vocab, history, bias, masks)
    Call(gpu_lib, torch, case).check()
    Call(gpu_lib, torch, case, logits=False).check()


def test_many_rows(gpu_lib, torch):
    Call(gpu_lib, torch, make(1, 200, 20000, 300, 20, 0.3)).check()


def test_a_vocabulary_of_several_passes(gpu_lib, torch):
    """slices longer than the counts that a block holds at a time"""
    Call(gpu_lib, torch, make(2, 3, 500_003, 5000, 1024, 0.4)).check()


@pytest.mark.parametrize("rows", [3, 33])
@pytest.mark.parametrize("history,bias", [(2560, 0), (2561, 0), (1536, 1024), (1537, 1024), (1536, 0), (1537, 0), (512, 1024), (513, 1024), (512, 1)])
def test_lists_where_the_table_ends(gpu_lib, torch, rows, history, bias):
    Call(gpu_lib, torch, make(history, rows, 40000, history, bias, 0.5)).check()


def test_as_many_rows_as_a_call_takes(gpu_lib, torch):
    case = make(5, 65535, 70, params=False)
    c = Call(gpu_lib, torch, case)
    c.call.run()
    torch.cuda.synchronize()
    assert (c.tokens.cpu().numpy() == case["logits"].argmax(1)).all() and (c.best.cpu().numpy() == case["logits"].max(1)).all()
    assert (c.out.cpu().numpy() == case["logits"]).all() and (c.status.cpu().numpy() == 0).all()


def test_longest_lists(gpu_lib, torch):
    case = make(3, 2, 5000, 65535, 1024, None)
    case["history"][1, :] = 4321                     # one token counts 65,535 times
    case["history_len"][1] = 65535
    case["bias_tokens"][1, :] = 17
    case["bias_values"][1, :] = (1 << 31) - 1        # sums beyond 32 bits
    case["bias_len"][1] = 1024
    case["params"][1] = [32768, 3, 2]
    Call(gpu_lib, torch, case).check()


def test_extreme_values(gpu_lib, torch):
    g = np.random.default_rng(4)
    case = make(4, 8, 3001, 900, 60, 0.7)
    edge = np.array([LOWEST, LOWEST + 1, -(1 << 30), -1, 0, 1, (1 << 30), (1 << 31) - 2, (1 << 31) - 1])
    case["logits"] = edge[g.integers(0, len(edge), (8, 3001))].astype(np.int32)
    case["params"][:, 0] = [1, 2, 32767, 32768, 32769, (1 << 31) - 1, 3, 65536]
    case["params"][:, 1] = [LOWEST, (1 << 31) - 1, 0, 1, -1, LOWEST, 7, 0]
    case["params"][:, 2] = [(1 << 31) - 1, LOWEST, 0, 1, -1, 5, LOWEST, (1 << 31) - 1]
    Call(gpu_lib, torch, case).check()


def test_ties_go_to_the_lowest_index(gpu_lib, torch):
    case = make(5, 6, 40000, params=False)
    case["logits"][:] = np.minimum(case["logits"], 99999)
    for r, at in enumerate(([39999], [0, 39999], [4, 5, 6, 7], [20000, 19999], [31999, 32000, 32001], [8191, 8192])):
        case["logits"][r, at] = 100000
    c = Call(gpu_lib, torch, case)
    c.check()
    assert c.tokens.tolist() == [39999, 0, 4, 19999, 31999, 8191]


def test_nothing_allowed(gpu_lib, torch):
    case = make(6, 3, 9000, masks=0.5)
    case["mask_page"][:] = [4, 0, -1]
    case["logits"][2] = LOWEST
    c = Call(gpu_lib, torch, case)
    c.check()
    assert c.tokens[0] == -2 and c.tokens[2] == -2 and c.best[2] == LOWEST and c.tokens[1] >= 0


def test_refused_rows_leave_the_others(gpu_lib, torch):
    case = make(7, 9, 20001, 50, 20, 0.5)
    case["mask_page"][:] = [-1, -5, 0, 1, 5, 2, 3, 0, 1]
    case["params"][1, 0] = 0
    case["params"][2, 0] = -3
    case["history_len"][3] = 51
    case["history_len"][5] = -1
    case["bias_len"][6] = 21
    case["bias_len"][7] = -1
    Call(gpu_lib, torch, case).check({1: 20, 2: 20, 3: 7, 4: 101, 5: 7, 6: 7, 7: 7})


@pytest.mark.parametrize("shift", [0, 1, 2, 3])
def test_strided_and_unaligned_rows_and_in_place(gpu_lib, torch, shift):
    case = make(8, 5, 4099, 100, 10, 0.5)
    c = Call(gpu_lib, torch, case)
    wide = torch.full((5, 4099 + 11), 7, dtype=torch.int32, device="cuda")
    logits = wide[:, shift:shift + 4099]
    logits.copy_(c.d["logits"])
    out = torch.full((5, 4099 + 6), 8, dtype=torch.int32, device="cuda")
    masks = torch.zeros((5, 600), dtype=torch.uint8, device="cuda")
    masks[:, 3:3 + 513] = c.d["masks"]
    args = dict(c.d, logits=logits, masks=masks[:, 3:3 + 513], out_tokens=c.tokens, out_best=c.best, row_status=c.status)
    abi.Pick(gpu_lib, out_logits=out[:, 2:2 + 4099], **args).run()
    torch.cuda.synchronize()
    c.out.copy_(out[:, 2:2 + 4099])
    c.compare()
    assert (out[:, :2] == 8).all() and (out[:, 4101:] == 8).all()
    abi.Pick(gpu_lib, out_logits=logits, **args).run()
    torch.cuda.synchronize()
    c.out.copy_(logits)
    c.compare()
    assert (wide[:, :shift] == 7).all() and (wide[:, shift + 4099:] == 7).all()


def test_offsets_beyond_32_bits(gpu_lib, torch):
    rows, vocab, stride = 5, 151936, 300_000_000      # the fifth row begins 4.8 GB behind the first
    case = make(9, rows, vocab, 100, 4)
    c = Call(gpu_lib, torch, case, logits=False)
    big = torch.empty(4 * stride + vocab, dtype=torch.int32, device="cuda")
    logits = big.as_strided((rows, vocab), (stride, 1))
    logits.copy_(c.d["logits"])
    abi.Pick(gpu_lib, out_tokens=c.tokens, out_best=c.best, row_status=c.status, **dict(c.d, logits=logits)).run()
    torch.cuda.synchronize()
    c.compare()


def test_captured_and_replayed(gpu_lib, torch):
    cases = [make(s, 7, 33000, 200, 9, 0.5) for s in (10, 11, 12)]
    c = Call(gpu_lib, torch, cases[0])
    c.check()
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.stream(stream):
        with torch.cuda.graph(graph, stream=stream):
            c.call.run()
    for case in cases[1:]:
        for k, v in case.items():
            c.d[k].copy_(torch.from_numpy(v))
        c.case = case
        graph.replay()
        torch.cuda.synchronize()
        c.compare()


def test_calls_on_two_streams(gpu_lib, torch):
    calls = [Call(gpu_lib, torch, make(20 + i, 30, 50000, 100, 10, 0.5)) for i in range(2)]
    streams = [torch.cuda.Stream() for _ in calls]
    torch.cuda.synchronize()
    for _ in range(20):
        for c, s in zip(calls, streams):
            c.call.run(s.cuda_stream)
    torch.cuda.synchronize()
    for c in calls:
        c.compare()


@pytest.mark.parametrize("rows,vocab,exchange", [(3, 100000, 0), (3, 100000, 1), (200, 30000, 1)])
def test_a_wait_that_runs_out(gpu_lib, torch, rows, vocab, exchange):
    """block 0 waits for more than its peers send, or than its copy of logits brings: its row is reported, the next call is right"""
    arm = gpu_lib.dll.sslm_b200_debug_withhold_exchange
    arm.argtypes = [C.c_int32, C.c_int32]
    assert arm(7, 2) == abi.ST["SSLM_INVALID_ARGUMENT"]
    c = Call(gpu_lib, torch, make(30, rows, vocab, 10, 0, None))
    try:
        assert arm(7, exchange) == 0
        c.call.run()
        torch.cuda.synchronize()
    finally:
        arm(-1, 0)
    assert c.status.tolist() == [100] + [0] * (rows - 1)
    c.check()


def test_a_block_by_itself_has_no_peers_to_outlast(gpu_lib, torch):
    """a row of one block, its copy late: a wait for the copy (0.25 s) and one more for what is under way, and no third for words of a peer"""
    import time
    arm = gpu_lib.dll.sslm_b200_debug_withhold_exchange
    arm.argtypes = [C.c_int32, C.c_int32]
    c = Call(gpu_lib, torch, make(33, 200, 9000))
    c.check()
    try:
        assert arm(7, 1) == 0
        begun = time.perf_counter()
        c.call.run()
        torch.cuda.synchronize()
        took = time.perf_counter() - begun
    finally:
        arm(-1, 0)
    assert c.status.tolist() == [100] + [0] * 199
    assert 0.25 <= took < 0.75
    c.check()


def test_no_rows(gpu_lib, torch):
    c = Call(gpu_lib, torch, make(31, 2, 50))
    c.call.args.rows = 0
    c.call.run()
    torch.cuda.synchronize()
    assert c.tokens.tolist() == [55, 55]


@pytest.mark.parametrize("logits", [False, True])
@pytest.mark.parametrize("rows,vocab,history", [(160, 600_001, 0), (160, 60_000, 3000), (1, 600_001, 0)])
def test_a_copy_that_is_late_ahead_of_other_chunks_and_passes(gpu_lib, torch, rows, vocab, history, logits):
    """more chunks than places, and passes behind the one whose copy is late: its row is reported, the others and the next call are right"""
    arm = gpu_lib.dll.sslm_b200_debug_withhold_exchange
    arm.argtypes = [C.c_int32, C.c_int32]
    case = make(32, rows, vocab, history, 0, None)
    c = Call(gpu_lib, torch, case, logits=logits)
    try:
        assert arm(7, 1) == 0
        c.call.run()
        torch.cuda.synchronize()
    finally:
        arm(-1, 0)
    assert c.status.tolist() == [100] + [0] * (rows - 1)
    some = sorted({1, rows // 2, rows - 1} - {0, rows})
    for r in some:
        assert (int(c.tokens[r]), int(c.best[r])) == picked(row_of(case, r))
    c.call.run()
    torch.cuda.synchronize()
    assert c.status.tolist() == [0] * rows
    for r in [0] + some:
        assert (int(c.tokens[r]), int(c.best[r])) == picked(row_of(case, r))
        if logits:
            assert (c.out[r].cpu().numpy() == row_of(case, r)).all()


@pytest.mark.parametrize("rows,vocab", [(6, 20001), (6, 900)])
def test_only_minus_one_says_no_mask(gpu_lib, torch, rows, vocab):
    case = make(34, rows, vocab, 50, 20, 0.5)
    case["mask_page"][:] = [-2, -1, 3, LOWEST, 0, 5]
    Call(gpu_lib, torch, case).check({0: 101, 3: 101, 5: 101})
