"""sslm_b200_qkv_site_resident: projections to codes of q, softmax constants and pages of K and V, against its definition in whole numbers."""
import numpy as np
import pytest

from superslm_b200 import abi
from tests.support.resident_more import PAGE, site_case, site_rows

pytestmark = pytest.mark.gpu


@pytest.fixture()
def torch():
    t = pytest.importorskip("torch")
    assert t.cuda.is_available()
    t.cuda.set_device(0)
    return t


class Call:
    def __init__(self, lib, torch, case, parts="qkv", **more):
        self.torch, self.case, self.parts = torch, case, parts
        H, KVH, hd = case["shape"]
        rows = len(case["wide"])
        self.d = {k: torch.from_numpy(v).cuda() if isinstance(v, np.ndarray) else v for k, v in case.items()}
        self.q_codes = torch.full((rows, H, hd), 55, dtype=torch.int8, device="cuda")
        self.q_scales = torch.full((rows, 2), 55, dtype=torch.int64, device="cuda")
        self.consts = torch.full((rows, KVH, 3), 55, dtype=torch.int64, device="cuda")
        self.saturations = torch.full((rows,), 55, dtype=torch.int32, device="cuda")
        self.status = torch.full((rows,), 77, dtype=torch.int32, device="cuda")
        d = self.d
        q, k, v = (d["wide"][:, a * hd:b * hd].view(rows, b - a, hd) for a, b in ((0, H), (H, H + KVH), (H + KVH, H + 2 * KVH)))
        args = dict(q=q if "q" in parts else None, k=k if "k" in parts else None, v=v if "k" in parts else None, in_scales=d["in_scales"], positions=d["positions"],
                    cos=d["cos"], sin=d["sin"], kv=d["kv"], pages=d["pages"], places=d["places"], table_of=d["table_of"], q_site=case["q_site"], khead=d["khead"],
                    k_landing=d["k_landing"], v_landing=d["v_landing"], q_gain=d["q_gain"], k_gain=d["k_gain"], gain_shift=case["q_shift"], k_gain_shift=case["k_shift"],
                    halves=case["halves"], saturations=self.saturations, row_status=self.status)
        if "q" in parts:
            args.update(q_codes=self.q_codes, q_scales=self.q_scales, consts=self.consts)
        self.args = dict(args, **more)
        self.call = abi.QkvSite(lib, **self.args)

    def check(self, refused=(), only=None):
        self.call.run()
        self.torch.cuda.synchronize()
        self.compare(refused, only)

    def compare(self, refused=(), only=None):
        case = self.case
        H, KVH, hd = case["shape"]
        got = [t.cpu().numpy() for t in (self.q_codes, self.q_scales, self.consts, self.saturations, self.status)]
        kv, before = self.d["kv"].cpu().numpy(), case["kv"].copy()
        rows = [r for r in (range(len(case["wide"])) if only is None else only) if r not in refused]
        want = site_rows(case, rows)
        for r in refused:
            assert got[4][r] == refused[r] and (got[0][r] == 55).all() and (got[1][r] == 55).all() and (got[2][r] == 55).all() and got[3][r] == 55, r
        touched = set()
        for r in rows:
            codes, scale, consts, sat, K, V = want[r]
            if "q" in self.parts:
                assert (got[0][r] == codes).all(), (r, np.argwhere(got[0][r] != codes)[:4])
                assert tuple(got[1][r]) == tuple(scale) and (got[2][r] == consts).all(), (r, got[1][r], scale, got[2][r], consts)
                assert got[4][r] == (0 if (consts[:, 0] > 0).all() else 23)
            else:
                assert (got[0][r] == 55).all() and got[4][r] == 0
            if "k" in self.parts:
                page, slot = case["pages"][case["table_of"][r], case["places"][r] // PAGE], case["places"][r] % PAGE
                assert (kv[:, 0, page].reshape(KVH, PAGE, hd)[:, slot] == K).all(), r
                assert (kv[:, 1, page].reshape(KVH, hd, PAGE)[:, :, slot] == V).all(), r
                assert got[3][r] == sat
                before[:, 0, page].reshape(KVH, PAGE, hd)      # (views of a copy do not write through: below)
                for h in range(KVH):
                    before[h, 0, page, slot * hd:(slot + 1) * hd] = K[h]
                    before[h, 1, page, slot::PAGE] = V[h]
                touched.add((page, slot))
        if only is None:
            assert (kv == before).all()                       # nothing else of the pool


@pytest.mark.parametrize("shape", [(14, 2, 64), (12, 2, 128), (16, 2, 128), (4, 2, 32), (8, 8, 64), (5, 1, 32), (1, 1, 128), (3, 3, 64)])
@pytest.mark.parametrize("norm,halves,part", [("", False, 1), ("", True, 1), ("qk", False, 2), ("k", True, 2), ("q", True, 1)])
def test_shapes(gpu_lib, torch, shape, norm, halves, part):
    Call(gpu_lib, torch, site_case(1, shape, 5, rotary=shape[2] // part, halves=halves, norm=norm)).check()


@pytest.mark.parametrize("rotary", [0, 8, 24, 40, 56, 64])
@pytest.mark.parametrize("halves", [False, True])
def test_part_of_a_head(gpu_lib, torch, rotary, halves):
    Call(gpu_lib, torch, site_case(2, (2, 1, 64), 3, rotary=rotary, halves=halves)).check()


@pytest.mark.parametrize("rows", [1, 2, 511, 513])
def test_rows_of_a_few_sequences(gpu_lib, torch, rows):
    """up to a row for every SM, and more"""
    c = Call(gpu_lib, torch, site_case(3, (2, 1, 32), rows, positions=400, tables=min(rows, 3), norm="k"))
    c.check(only=None if rows < 600 else range(0, rows, 17))


@pytest.mark.parametrize("shape", [(40, 8, 128), (60, 30, 64), (96, 80, 128), (254, 1, 128)])
def test_wide_rows(gpu_lib, torch, shape):
    """up to 32,768 elements: four and sixteen quads a thread"""
    Call(gpu_lib, torch, site_case(4, shape, 2, norm="k")).check()


@pytest.mark.parametrize("quads", [1024, 1056, 2048, 2080, 4096, 4128, 8192])
def test_where_the_threads_of_a_row_change(gpu_lib, torch, quads):
    Call(gpu_lib, torch, site_case(15, (quads // 32 - 2, 1, 128), 1)).check()


def by_hundreds(gpu_lib, torch, case):
    """the same rows in calls of 100, a block a row"""
    whole, parts = Call(gpu_lib, torch, case), []
    whole.call.run()
    kv = torch.from_numpy(case["kv"]).cuda()
    for r in range(0, len(case["wide"]), 100):
        cut = dict(case, **{k: case[k][r:r + 100] for k in ("wide", "in_scales", "positions", "places", "table_of")})
        parts.append(Call(gpu_lib, torch, cut, kv=kv))
        parts[-1].call.run()
    torch.cuda.synchronize()
    for name in ("q_codes", "q_scales", "consts", "saturations", "status"):
        assert torch.equal(getattr(whole, name), torch.cat([getattr(c, name) for c in parts])), name
    assert torch.equal(whole.d["kv"], kv)
    return whole


def many_rows(torch, seed, shape, more=5, first=3, **kind):
    """eight rows for every SM and a few more, enough for the form of many rows; three sequences' places run on from `first`, the other rows' are drawn"""
    rows = 8 * torch.cuda.get_device_properties(0).multi_processor_count + more
    case = site_case(seed, shape, rows, positions=512, tables=6, **kind)
    g = np.random.default_rng(seed)
    places = np.zeros(rows, dtype=np.int64)
    at = 0
    for s, n in enumerate((300, 211, rows - 511 - 400)):
        case["table_of"][at:at + n], places[at:at + n], at = s, np.arange(first, first + n), at + n
    case["table_of"][at:] = 3 + np.arange(400) % 3
    for s in range(3, 6):
        mine = np.flatnonzero(case["table_of"] == s)
        places[mine] = g.choice(512, len(mine), replace=False)
    assert places.max() < 512
    case["places"] = places.astype(np.int32)
    return case


@pytest.mark.parametrize("shape,norm,halves,part", [((14, 2, 64), "", False, 1), ((12, 2, 128), "", False, 1), ((12, 2, 128), "q", True, 2), ((4, 2, 32), "k", True, 1), ((5, 1, 32), "", True, 4),
                                                    ((1, 1, 128), "qk", False, 1), ((16, 2, 128), "", True, 1), ((16, 4, 128), "qk", False, 2), ((3, 3, 64), "", False, 1), ((27, 2, 128), "", False, 1)])
def test_many_rows(gpu_lib, torch, shape, norm, halves, part):
    case = many_rows(torch, 16, shape, rotary=shape[2] // part, halves=halves, norm=norm)
    c = by_hundreds(gpu_lib, torch, case)
    c.compare(only=[0, 1, 2, 3, 4, 298, 299, 300, 301, 510, 511, 800, len(case["wide"]) - 1])


@pytest.mark.parametrize("first,more", [(0, 0), (4, 1), (7, 8), (16, 13)])
def test_many_rows_that_begin_anywhere(gpu_lib, torch, first, more):
    by_hundreds(gpu_lib, torch, many_rows(torch, 17, (2, 1, 64), more=more, first=first))


@pytest.mark.parametrize("parts", ["q", "k"])
@pytest.mark.parametrize("norm", ["", "qk"])
def test_parts_of_many_rows(gpu_lib, torch, parts, norm):
    case = many_rows(torch, 18, (6, 2, 64), norm=norm)
    c = Call(gpu_lib, torch, case, parts)
    c.check(only=[0, 5, 9, 299, 300, 700, len(case["wide"]) - 1])
    c = Call(gpu_lib, torch, dict(case, cos=np.zeros((512, 0), dtype=np.int32), sin=np.zeros((512, 0), dtype=np.int32)), parts)      # (nothing is turned)
    c.check(only=[0, 5, 9, 299, 300, 700, len(case["wide"]) - 1])


@pytest.mark.parametrize("halves", [False, True])
def test_many_rows_of_ties(gpu_lib, torch, halves):
    """angles of whole eighths and landings by powers of two: a half is common, and a result out of range"""
    case = many_rows(torch, 19, (4, 2, 64), halves=halves, deviation=3000.0)
    g = np.random.default_rng(19)
    rows = len(case["wide"])
    case["cos"], case["sin"] = ((g.integers(-12, 13, case["cos"].shape) << 27).astype(np.int32) for _ in range(2))
    case["cos"][0], case["sin"][0] = -(1 << 31), (1 << 31) - 1
    case["positions"][::50] = 0
    case["in_scales"][:, 0] = 1 << 30
    for name in ("k_landing", "v_landing"):
        case[name][:] = 1 << 30, -50 + 6, 1 << 32
    case["in_scales"][:, 1] = -50 + g.integers(-2, 3, rows)
    c = by_hundreds(gpu_lib, torch, case)
    c.compare(only=[0, 1, 50, 77, 299, 300, 600, rows - 1])


def test_many_rows_with_values_at_the_ends(gpu_lib, torch):
    case = many_rows(torch, 20, (2, 1, 32))
    w = case["wide"]
    w[0], w[1], w[2], w[3], w[3, 5] = 0, -(1 << 31), (1 << 31) - 1, 0, 1
    w[4] = np.where(np.arange(128) % 2, 1 << 24, -(1 << 24) - 1)
    w[5], w[6] = 1 << 30, np.arange(128) - 64
    w[60:90] = np.random.default_rng(20).integers(-(1 << 31), 1 << 31, (30, 128))
    for r, (m, e) in {7: (1 << 30, 20), 8: ((1 << 31) - 1, -100), 9: (1 << 30, 60), 10: (1 << 30, 4096), 11: ((1 << 31) - 1, -4096), 61: (1 << 30, -60), 62: (1 << 30, -70)}.items():
        case["in_scales"][r] = m, e
    c = by_hundreds(gpu_lib, torch, case)
    c.compare(only=list(range(0, 13)) + list(range(58, 92)))
    case["k_landing"][0, 1], case["v_landing"][0, 1] = 1 << 40, -(1 << 62)
    c = by_hundreds(gpu_lib, torch, case)
    c.case = dict(case, k_landing=case["k_landing"].copy(), v_landing=case["v_landing"].copy())
    c.case["k_landing"][0, 1], c.case["v_landing"][0, 1] = 20000, -20000      # as far out of range, and a number that the definition can shift by
    c.compare(only=[0, 1, 4, 9, 70])
    case["k_landing"][0, 2], case["v_landing"][0, 2] = 0, (1 << 40) + 1
    by_hundreds(gpu_lib, torch, case)


def test_many_rows_some_refused_and_left_out(gpu_lib, torch):
    case = many_rows(torch, 21, (4, 2, 64))
    n = len(case["wide"])
    case["positions"][1] = -1
    case["positions"][2] = -2
    case["positions"][3] = 512
    case["places"][4] = 512
    case["places"][5] = -1
    case["table_of"][6] = 6
    case["table_of"][7] = -1
    case["pages"][3, case["places"][np.flatnonzero(case["table_of"] == 3)[-1]] // PAGE] = -1
    case["in_scales"][10, 0] = (1 << 30) - 1
    case["in_scales"][11, 0] = 1 << 31
    case["in_scales"][12, 1] = 4097
    case["positions"][16:24] = -1                             # a tile of padding
    case["positions"][n - 1] = -1
    c = by_hundreds(gpu_lib, torch, case)
    status = c.status.cpu().numpy()
    assert list(status[:13]) == [0, 0, 7, 7, 7, 7, 101, 101, 0, 0, 20, 20, 20] and (status[16:24] == 0).all() and status[n - 1] == 0
    assert 101 in status[511:] and (c.q_codes[16:24] == 55).all() and (c.saturations[1:8] == 55).all()
    c.compare(only=[0, 8, 9, 13, 15, 24])
    c = Call(gpu_lib, torch, dict(case, positions=np.full(n, 512, dtype=np.int32)))
    c.call.run()
    torch.cuda.synchronize()
    assert (c.status == 7).all() and (c.q_codes == 55).all()


@pytest.mark.parametrize("parts", ["q", "k"])
@pytest.mark.parametrize("norm", ["", "qk"])
def test_parts(gpu_lib, torch, parts, norm):
    Call(gpu_lib, torch, site_case(5, (6, 2, 64), 4, norm=norm), parts).check()


def test_values_at_the_ends(gpu_lib, torch):
    case = site_case(6, (2, 1, 32), 12, norm="")
    case["wide"][0] = 0
    case["wide"][1] = -(1 << 31)
    case["wide"][2] = (1 << 31) - 1
    case["wide"][3, :] = 0
    case["wide"][3, 5] = 1
    case["wide"][4] = np.where(np.arange(128) % 2, 1 << 24, -(1 << 24) - 1)
    case["wide"][5] = 1 << 30
    case["wide"][6] = np.arange(128) - 64
    case["in_scales"][7] = 1 << 30, 20                        # lands far outside
    case["in_scales"][8] = (1 << 31) - 1, -100                # lands on zero
    case["in_scales"][9] = 1 << 30, 60                        # a negative shift
    case["in_scales"][10] = 1 << 30, 4096
    case["in_scales"][11] = (1 << 31) - 1, -4096
    c = Call(gpu_lib, torch, case)
    c.check()
    normal = dict(case, q_gain=np.full(32, 32767, dtype=np.int16), k_gain=np.full(32, -32768, dtype=np.int16))
    for q_shift, k_shift in ((1, 62), (23, 1), (40, 24)):
        Call(gpu_lib, torch, dict(normal, q_shift=q_shift, k_shift=k_shift)).check()


def test_a_norm_does_not_know_its_scale(gpu_lib, torch):
    """heads times a power of two are the same codes, and they are near the norm in floating point"""
    case = site_case(7, (4, 1, 128), 6, norm="qk", deviation=900.0)
    case["wide"][1:] = case["wide"][0]
    for r in range(1, 6):
        case["wide"][r] <<= 3 * r
    case["positions"][:] = 5
    c = Call(gpu_lib, torch, case)
    c.check()
    assert (c.q_codes == c.q_codes[:1]).all()
    x = case["wide"][0, :512].reshape(4, 128).astype(np.float64)
    flat = dict(case, cos=np.full_like(case["cos"], 1 << 30), sin=np.zeros_like(case["sin"]))
    c = Call(gpu_lib, torch, flat)
    c.check()
    exact = x / np.sqrt((x * x).mean(1, keepdims=True)) * case["q_gain"] / 2.0 ** (case["q_shift"] - 15)
    # half a code, and what u's rounding (2^-16 of it), the root's (2^-22) and the reciprocal's (2^-26) move one of 127 by
    assert np.abs(c.q_codes[0].cpu().numpy() - np.clip(exact, -127, 127)).max() <= 0.5 + 9000 / 2.0 ** 24 + 127 * 2.0 ** -21


def test_no_constants(gpu_lib, torch):
    case = site_case(8, (4, 2, 32), 4)
    case["khead"][1] = (1 << 30, 60)                          # a scale so coarse that ln 2 is less than one unit
    Call(gpu_lib, torch, case).check()
    case["khead"][0] = (1 << 30, -200)
    Call(gpu_lib, torch, case).check()


def test_refused_rows_and_rows_left_out(gpu_lib, torch):
    case = site_case(9, (4, 2, 64), 14)
    case["positions"][1] = -1                                 # a padded row
    case["positions"][2] = -2
    case["positions"][3] = 64
    case["places"][4] = 64
    case["places"][5] = -1
    case["table_of"][6] = 14
    case["table_of"][7] = -1
    case["pages"][8, case["places"][8] // PAGE] = -1
    case["pages"][9, case["places"][9] // PAGE] = case["kv"].shape[2]
    case["in_scales"][10, 0] = (1 << 30) - 1
    case["in_scales"][11, 0] = 1 << 31
    case["in_scales"][12, 1] = 4097
    Call(gpu_lib, torch, case).check({1: 0, 2: 7, 3: 7, 4: 7, 5: 7, 6: 101, 7: 101, 8: 101, 9: 101, 10: 20, 11: 20, 12: 20})


def test_places_are_positions_and_tables_rows(gpu_lib, torch):
    case = site_case(10, (4, 2, 64), 6)
    case["places"], case["table_of"] = case["positions"], np.arange(6, dtype=np.int32)
    Call(gpu_lib, torch, case, places=None, table_of=None).check()


def test_strided_rows(gpu_lib, torch):
    c = Call(gpu_lib, torch, site_case(11, (4, 2, 64), 5))
    q = torch.full((5, 700), 9, dtype=torch.int32, device="cuda")
    k, v = (torch.full((5, 140), 9, dtype=torch.int32, device="cuda") for _ in range(2))
    codes = torch.full((5, 300), 3, dtype=torch.int8, device="cuda")
    q[:, 400:656] = c.d["wide"][:, :256]
    k[:, 12:140] = c.d["wide"][:, 256:384]
    v[:, :128] = c.d["wide"][:, 384:]
    pages = torch.full((5, 9), -1, dtype=torch.int32, device="cuda")
    pages[:, 2:6] = c.d["pages"]
    args = dict(c.args, q=q[:, 400:656].view(5, 4, 64), k=k[:, 12:140].view(5, 2, 64), v=v[:, :128].view(5, 2, 64), q_codes=codes[:, 20:276].view(5, 4, 64), pages=pages[:, 2:6])
    abi.QkvSite(gpu_lib, **args).run()
    torch.cuda.synchronize()
    c.q_codes.copy_(codes[:, 20:276].view(5, 4, 64))
    c.compare()
    assert (codes[:, :20] == 3).all() and (codes[:, 276:] == 3).all()


def test_captured_and_replayed(gpu_lib, torch):
    cases = [site_case(s, (4, 2, 64), 7, norm="k") for s in (12, 13)]
    c = Call(gpu_lib, torch, cases[0])
    c.check()
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.stream(stream):
        with torch.cuda.graph(graph, stream=stream):
            c.call.run()
    case = dict(cases[1], q_site=cases[0]["q_site"])
    for k, v in case.items():
        if isinstance(v, np.ndarray):
            c.d[k].copy_(torch.from_numpy(v))
    c.case = case
    graph.replay()
    torch.cuda.synchronize()
    c.compare()


def test_pages_beyond_32_bits(gpu_lib, torch):
    case = site_case(14, (2, 1, 128), 3)
    c = Call(gpu_lib, torch, case)
    far = 1_200_000                                           # K pages of 2 KB: the last one 2.4 GB behind the first, V's another 2.4
    kv = torch.zeros((1, 2, far, PAGE * 128), dtype=torch.int8, device="cuda")
    last = torch.arange(far - case["kv"].shape[2], far, device="cuda")
    kv[:, :, last] = c.d["kv"]
    pages = c.d["pages"] + (far - case["kv"].shape[2])
    abi.QkvSite(gpu_lib, **dict(c.args, kv=kv, pages=pages)).run()
    torch.cuda.synchronize()
    c.d["kv"].copy_(kv[:, :, last])
    c.compare()
