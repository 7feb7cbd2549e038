"""sslm_b200_sample_resident: a token drawn with temperature, top-k, top-p and min-p, against its definition in whole numbers."""
import ctypes as C
import math

import numpy as np
import pytest

from superslm_b200 import abi
from tests.support.resident_more import LOWEST, drawn

pytestmark = pytest.mark.gpu
NAT = 36000.0


@pytest.fixture()
def torch():
    t = pytest.importorskip("torch")
    assert t.cuda.is_available()
    t.cuda.set_device(0)
    return t


def make(seed, rows, vocab, top_k=0, top_p=1.0, min_p=0.0, spread=2.2, allowed=1.0, logits=None):
    g = np.random.default_rng(seed)
    if logits is None:
        logits = g.normal(0, spread * NAT, (rows, vocab))
        for r in range(rows):
            logits[r, g.integers(0, vocab, 30)] += g.uniform(3, 10, 30) * NAT
        logits = np.rint(logits)
    logits = np.array(logits, dtype=np.int32, order="C")
    if allowed < 1:
        logits[g.random((rows, vocab)) >= allowed] = LOWEST
    params = np.array([abi.sample_params(1 / NAT, g.uniform(0.5, 1.4), top_k, top_p, min_p) for _ in range(rows)], dtype=np.int32)
    return dict(logits=logits, params=params, draws=g.integers(0, 1 << 31, rows).astype(np.int32))


class Call:
    def __init__(self, lib, torch, case, **more):
        self.torch, self.case = torch, case
        self.d = {k: torch.from_numpy(v).cuda() for k, v in case.items()}
        rows = len(case["draws"])
        self.tokens, self.kept, self.status = (torch.full((rows,), 55, dtype=torch.int32, device="cuda") for _ in range(3))
        self.mass = torch.full((rows, 2), 55, dtype=torch.int64, device="cuda")
        self.outputs = dict(out_tokens=self.tokens, out_mass=self.mass, out_kept=self.kept, row_status=self.status)
        self.call = abi.Sample(lib, **dict(self.d, **dict(self.outputs, **more)))

    def check(self, refused=()):
        self.call.run()
        self.torch.cuda.synchronize()
        self.compare(refused)

    def compare(self, refused=()):
        tokens, mass, kept, status = (t.cpu().numpy() for t in (self.tokens, self.mass, self.kept, self.status))
        for r in range(len(tokens)):
            if r in refused:
                assert status[r] == refused[r] and tokens[r] == kept[r] == 55 and (mass[r] == 55).all(), r
                continue
            want = drawn(self.case["logits"][r], *(int(v) for v in self.case["params"][r]), int(self.case["draws"][r]))
            assert (tokens[r], mass[r, 0], mass[r, 1], kept[r]) == want and status[r] == 0, (r, tokens[r], mass[r], kept[r], want)


WIDE = "a tenth of all tokens"      # more than the first list has
LIMITS = [dict(), dict(top_k=1), dict(top_k=50), dict(top_p=0.9), dict(min_p=0.05), dict(top_k=40, top_p=0.95), dict(top_k=900, top_p=0.7, min_p=0.001), dict(top_p=0.5, min_p=0.3)]


@pytest.mark.parametrize("vocab", [1, 2, 5, 127, 129, 500, 2049, 4097, 8191, 32003])
@pytest.mark.parametrize("limits", LIMITS)
def test_sizes(gpu_lib, torch, vocab, limits):
    Call(gpu_lib, torch, make(1, 3, vocab, **limits)).check()


@pytest.mark.parametrize("rows,vocab", [(1, 151936), (5, 151936), (20, 70001), (64, 40000), (160, 20001), (300, 9001)])
@pytest.mark.parametrize("limits", LIMITS)
def test_every_number_of_blocks(gpu_lib, torch, rows, vocab, limits):
    Call(gpu_lib, torch, make(2, rows, vocab, **limits)).check()


@pytest.mark.parametrize("rows,vocab", [(1, 151936), (3, 40009), (30, 60000), (90, 30001), (200, 40000)])
@pytest.mark.parametrize("top_p,spread,min_p", [(0.5, 4.0, 0.0), (0.9, 4.0, 0.0), (0.9, 3.0, 0.00001), (0.99, 2.5, 0.0), (0.9, 0.1, 0.0), (0.3, 0.01, 0.9), (0.99999, 3.0, 0.0), (0.9, 9.0, 0.0)])
def test_what_top_p_keeps_is_long(gpu_lib, torch, rows, vocab, top_p, spread, min_p):
    """temperatures that spread the weights: a window around the end of what is kept, behind thousands of tokens"""
    g = np.random.default_rng(16)
    logits = np.rint(g.normal(0, spread * NAT, (rows, vocab)))
    case = make(16, rows, vocab, top_p=top_p, min_p=min_p, logits=logits)
    Call(gpu_lib, torch, case).check()


@pytest.mark.parametrize("rows,vocab", [(1, 1 << 20), (2, 300001), (200, 262000)])
@pytest.mark.parametrize("limits", [dict(), dict(top_k=30, top_p=0.9)])
def test_long_rows(gpu_lib, torch, rows, vocab, limits):
    case = make(3, min(rows, 2), vocab, **limits)
    if rows > 2:      # (the definition takes its time)
        case = {k: np.resize(v, (rows,) + v.shape[1:]) for k, v in case.items()}
    c = Call(gpu_lib, torch, case)
    c.call.run()
    torch.cuda.synchronize()
    for t in (c.tokens, c.mass, c.kept, c.status):
        assert (t.view(-1, 2 if rows > 1 else 1, *t.shape[1:]) == t[:2 if rows > 1 else 1]).all()
    c.case = {k: v[:2] for k, v in case.items()}
    c.tokens, c.mass, c.kept, c.status = (t[:2] for t in (c.tokens, c.mass, c.kept, c.status))
    c.compare()


@pytest.mark.parametrize("limits", LIMITS + [dict(top_k=20000), dict(top_p=0.9999)])
@pytest.mark.parametrize("kind", ["equal", "two values", "rising", "falling", "flat"])
@pytest.mark.parametrize("rows,vocab", [(2, 30011), (170, 12001)])
def test_lists_that_do_not_do(gpu_lib, torch, kind, limits, rows, vocab):
    """many equal logits, logits in order, and a temperature at which thousands are kept: more tokens than a list holds, or fewer than asked for"""
    v = np.arange(vocab)
    g = np.random.default_rng(4)
    x = {"equal": np.full(vocab, 777), "two values": np.where(g.random(vocab) < 0.3, 5000, -900), "rising": 3 * v, "falling": -3 * v, "flat": g.integers(-20000, 20000, vocab)}[kind]
    Call(gpu_lib, torch, make(5, rows, vocab, logits=np.broadcast_to(x, (rows, vocab)), **limits)).check()


@pytest.mark.parametrize("limits", LIMITS)
def test_masked_tokens(gpu_lib, torch, limits):
    case = make(6, 9, 60001, allowed=0.02, **limits)
    case["logits"][1] = LOWEST                                  # nothing is allowed
    case["logits"][2] = LOWEST
    case["logits"][2, 59999] = LOWEST + 1                       # one token, the lowest logit there is
    case["logits"][3, :50000] = LOWEST                          # allowed tokens in the last blocks alone
    case["logits"][4, 1000:] = LOWEST
    case["logits"][4, 0] = (1 << 31) - 1
    case["logits"][5] = LOWEST
    case["logits"][5, 20000:34000] = 5                          # more equal ones than a list holds
    c = Call(gpu_lib, torch, case)
    c.check()
    assert c.tokens[1] == -2 and c.kept[1] == 0 and c.tokens[2] == 59999


@pytest.mark.parametrize("slope,cut", [(0, 0), (1, 63), (1, 0), ((1 << 31) - 1, 0), ((1 << 31) - 1, 33), ((1 << 31) - 1, 34), (1 << 30, 62), (1 << 24, 0), ((1 << 29) - 1, 10), (77, 3)])
def test_slopes(gpu_lib, torch, slope, cut):
    g = np.random.default_rng(7)
    case = make(7, 6, 5003, top_p=0.9)
    case["logits"][0, :] = g.integers(LOWEST, -LOWEST, 5003)
    case["logits"][1, :] = g.integers(0, 5, 5003)
    case["params"][:, 0], case["params"][:, 1] = slope, cut
    case["params"][3:, 2], case["params"][3:, 3] = 3, 1 << 30
    case["params"][5, 2] = 0
    Call(gpu_lib, torch, case).check()


@pytest.mark.parametrize("rows,vocab", [(2, 151936), (70, 33001), (150, 40000)])
@pytest.mark.parametrize("temperature", [1e-6, 1e-3, 0.03, 30.0, 1e5])
@pytest.mark.parametrize("limits", [dict(top_k=50, top_p=0.95), dict(top_k=400), dict(top_k=900, min_p=0.01), dict(top_p=0.9), dict()])
def test_steep_and_flat(gpu_lib, torch, rows, vocab, temperature, limits):
    """fewer tokens have a weight than top-k asks for, or all have nearly the same"""
    case = make(21, rows, vocab, **limits)
    case["params"][:] = [abi.sample_params(1 / NAT, temperature, **limits) for _ in range(rows)]
    case["logits"][1] = np.arange(vocab) % 7 * 1000
    Call(gpu_lib, torch, case).check()


def test_draws_and_limits_at_their_ends(gpu_lib, torch):
    case = make(8, 8, 4099)
    case["draws"][:4] = 0, (1 << 31) - 1, 1, 1 << 30
    case["params"][4, 2:] = (1 << 31) - 1, 1, 1 << 30
    case["params"][5, 2:] = 4099, 1 << 30, 0
    case["params"][6, 2:] = 4098, (1 << 30) - 1, 1
    case["params"][7, 2:] = 0, 1, 0
    case["draws"][4:] = (1 << 31) - 1
    c = Call(gpu_lib, torch, case)
    c.check()
    assert c.kept[4] == 1 and c.kept[7] == 1


def test_refused_rows_leave_the_others(gpu_lib, torch):
    case = make(9, 14, 20001, top_k=5)
    bad = [(1, 0, -1), (2, 1, -1), (3, 1, 64), (4, 2, -1), (5, 3, 0), (6, 3, (1 << 30) + 1), (7, 4, -1), (8, 4, (1 << 30) + 1), (9, 3, -5)]
    for r, i, v in bad:
        case["params"][r, i] = v
    case["draws"][10] = -1
    Call(gpu_lib, torch, case).check({r: 20 for r in range(1, 11)})


@pytest.mark.parametrize("shift", [0, 1, 2, 3])
@pytest.mark.parametrize("limits", [dict(), dict(top_k=20, top_p=0.9), dict(top_p=0.99999)])
def test_strided_and_unaligned_rows(gpu_lib, torch, shift, limits):
    c = Call(gpu_lib, torch, make(10, 5, 4099, **limits))
    wide = torch.full((5, 4099 + 11), (1 << 31) - 1, dtype=torch.int32, device="cuda")      # (what lies beside would win)
    wide[:, shift:shift + 4099] = c.d["logits"]
    abi.Sample(gpu_lib, **dict(c.d, logits=wide[:, shift:shift + 4099], **c.outputs)).run()
    torch.cuda.synchronize()
    c.compare()


def test_offsets_beyond_32_bits(gpu_lib, torch):
    rows, vocab, stride = 5, 50001, 300_000_000
    c = Call(gpu_lib, torch, make(11, rows, vocab, top_k=50, top_p=0.9))
    big = torch.empty(4 * stride + vocab, dtype=torch.int32, device="cuda")
    logits = big.as_strided((rows, vocab), (stride, 1))
    logits.copy_(c.d["logits"])
    abi.Sample(gpu_lib, **dict(c.d, logits=logits, **c.outputs)).run()
    torch.cuda.synchronize()
    c.compare()


def test_captured_and_replayed(gpu_lib, torch):
    cases = [make(s, 7, 33000, top_k=k, top_p=p) for s, k, p in ((12, 20, 0.9), (13, 0, 0.8), (14, 0, 1.0))]
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
    calls = [Call(gpu_lib, torch, make(20 + i, 30, 50000, top_k=30 * i, top_p=0.9)) for i in range(2)]
    streams = [torch.cuda.Stream() for _ in calls]
    torch.cuda.synchronize()
    for _ in range(20):
        for c, s in zip(calls, streams):
            c.call.run(s.cuda_stream)
    torch.cuda.synchronize()
    for c in calls:
        c.compare()


def test_probabilities(gpu_lib, torch):
    """w over the sum of all is the softmax: the polynomial is off by 3.4e-6 of a weight at most, the floor by 2^-31 of the largest, so a quotient by
    7e-6 of itself and 2^-31 of the largest (and the tokens beyond 2^-32 of it, 20,000 at most, by 5e-6)"""
    rng = np.random.default_rng(15)
    x = rng.normal(0, 2.0 * NAT, 20000).astype(np.int32)
    case = make(15, 400, 20000, logits=np.broadcast_to(x, (400, 20000)))
    case["params"][:] = abi.sample_params(1 / NAT, 0.8)
    c = Call(gpu_lib, torch, case)
    c.call.run()
    torch.cuda.synchronize()
    p = np.exp((x - x.max()) / NAT / 0.8)
    p /= p.sum()
    tokens, mass = c.tokens.cpu().numpy(), c.mass.cpu().numpy()
    got = mass[:, 0] / mass[:, 1]
    assert (np.abs(got - p[tokens]) <= 1.4e-5 * p[tokens] + 2.0 ** -31 * p.max()).all()
    # the draw is the inverse of the distribution function by index
    upto = np.cumsum(p)
    u = case["draws"] / 2.0 ** 31
    assert (upto[tokens] >= u - 1.4e-5).all() and (upto[tokens] - p[tokens] <= u + 1.4e-5).all()


@pytest.mark.parametrize("exchange,limits", [(0, dict()), (1, dict(top_k=40, top_p=0.9)), (2, dict(top_k=40, top_p=0.9)), (3, WIDE), (4, WIDE), (5, WIDE), (6, WIDE), (7, WIDE)])
def test_a_wait_that_runs_out(gpu_lib, torch, exchange, limits):
    """block 0 waits for more than its peers send: its row is reported, the others are right, and so is the next call"""
    arm = gpu_lib.dll.sslm_b200_debug_withhold_exchange
    arm.argtypes = [C.c_int32, C.c_int32]
    assert arm(8, 8) == abi.ST["SSLM_INVALID_ARGUMENT"]
    if limits is WIDE:
        case = make(30, 3, 100000, top_p=0.9, logits=np.random.default_rng(30).normal(0, 2.5 * NAT, (3, 100000)))
        case["params"][:, :2] = abi.sample_params(1 / NAT)[:2]
    else:
        case = make(30, 3, 100000, **limits)
    c = Call(gpu_lib, torch, case)
    try:
        assert arm(8, exchange) == 0
        c.call.run()
        torch.cuda.synchronize()
    finally:
        arm(-1, 0)
    assert c.status.tolist() == [100, 0, 0]
    c.check()
    if limits is WIDE:
        assert (c.kept > 4000).all()


def test_what_a_caller_leaves_out(gpu_lib, torch):
    c = Call(gpu_lib, torch, make(31, 4, 9000, top_k=9))
    for name in ("out_tokens", "out_mass", "out_kept"):
        abi.Sample(gpu_lib, **dict(c.d, **{name: c.outputs[name]})).run()
    c.status.zero_()
    torch.cuda.synchronize()
    c.compare()


def test_parameters():
    for scale, temperature in ((1 / NAT, 1.0), (1.0, 1.0), (1e-9, 2.0), (1e-25, 1.0), (1e6, 0.01)):
        slope, cut, top_k, top_p, min_p = abi.sample_params(scale, temperature, 7, 0.5, 0.25)
        assert 0 <= slope < 1 << 31 and 0 <= cut <= 63 and (top_k, top_p, min_p) == (7, 1 << 29, 1 << 28)
        octaves = scale / temperature / math.log(2) * 2.0 ** 24
        assert slope / 2.0 ** cut == pytest.approx(octaves, rel=2.0 ** -30) or octaves > 2.0 ** 30 or octaves < 2.0 ** -33
