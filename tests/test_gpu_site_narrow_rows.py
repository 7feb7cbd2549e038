"""The q/k/v site of rows so narrow that thousands of them take the form of many rows: the same as in calls of 100, a block a row, and as its definition."""
import numpy as np
import pytest

from tests.support.resident_more import PAGE, site_case
from tests.test_gpu_site import Call, by_hundreds

pytestmark = pytest.mark.gpu


@pytest.fixture()
def torch():
    t = pytest.importorskip("torch")
    assert t.cuda.is_available()
    t.cuda.set_device(0)
    return t


def many_rows(torch, seed, shape, quads=2048, more=5, first=3, **kind):
    """more than `quads` quads of elements for every SM; sequences of 300 and 211 rows in turn whose places run on from `first`, the last 400 rows' are drawn"""
    H, KVH, hd = shape
    rows = quads * torch.cuda.get_device_properties(0).multi_processor_count // ((H + 2 * KVH) * hd // 4) + more
    runs, at = [], 0
    while at < rows - 400:
        runs.append(min((300, 211)[len(runs) % 2], rows - 400 - at))
        at += runs[-1]
    case = site_case(seed, shape, rows, positions=512, tables=len(runs) + 3, **kind)
    places, at = np.zeros(rows, dtype=np.int64), 0
    for s, n in enumerate(runs):
        case["table_of"][at:at + n], places[at:at + n], at = s, np.arange(first, first + n), at + n
    case["table_of"][at:] = len(runs) + np.arange(400) % 3
    g = np.random.default_rng(seed)
    for s in range(len(runs), len(runs) + 3):
        mine = np.flatnonzero(case["table_of"] == s)
        places[mine] = g.choice(512, len(mine), replace=False)
    case["places"] = places.astype(np.int32)
    return case


def some(case):
    n = len(case["wide"])
    return [r for r in (0, 1, 2, 3, 4, 298, 299, 300, 301, 510, 511, 800, 1500) if r < n - 1] + [n - 1]


@pytest.mark.parametrize("shape,norm,halves,part", [((4, 2, 32), "", False, 1), ((4, 2, 32), "k", True, 1), ((5, 1, 32), "", True, 4), ((1, 1, 128), "", False, 1), ((3, 3, 64), "", False, 1),
                                                    ((2, 1, 32), "", True, 1), ((8, 8, 64), "k", False, 2)])
def test_landed(gpu_lib, torch, shape, norm, halves, part):
    case = many_rows(torch, 36, shape, rotary=shape[2] // part, halves=halves, norm=norm)
    by_hundreds(gpu_lib, torch, case).compare(only=some(case))


@pytest.mark.parametrize("shape,norm,halves,part", [((4, 2, 32), "qk", False, 1), ((1, 1, 128), "qk", False, 1), ((5, 1, 32), "q", True, 4), ((14, 2, 64), "qk", True, 2), ((12, 2, 128), "qk", True, 2),
                                                    ((16, 4, 128), "q", False, 1)])
def test_normed(gpu_lib, torch, shape, norm, halves, part):
    case = many_rows(torch, 37, shape, 5000, rotary=shape[2] // part, halves=halves, norm=norm)
    by_hundreds(gpu_lib, torch, case).compare(only=some(case))


@pytest.mark.parametrize("first,more", [(0, 0), (0, 1), (4, 2), (7, 8), (16, 13)])
def test_where_the_form_changes_and_places_that_begin_anywhere(gpu_lib, torch, first, more):
    by_hundreds(gpu_lib, torch, many_rows(torch, 38, (2, 1, 64), more=more, first=first))


@pytest.mark.parametrize("parts", ["q", "k"])
@pytest.mark.parametrize("norm", ["", "qk"])
def test_parts(gpu_lib, torch, parts, norm):
    H, KVH, hd = shape = (6, 2, 64)
    own = 2 * KVH if parts == "k" else H      # heads that the call has
    case = many_rows(torch, 39, shape, (5000 if "q" in norm and parts == "q" else 2048) * (H + 2 * KVH) // own + 1, norm=norm)
    only = [0, 5, 9, 299, 300, 700, len(case["wide"]) - 1]
    Call(gpu_lib, torch, case, parts).check(only=only)
    Call(gpu_lib, torch, dict(case, cos=np.zeros((512, 0), dtype=np.int32), sin=np.zeros((512, 0), dtype=np.int32)), parts).check(only=only)      # (nothing is turned)


@pytest.mark.parametrize("halves", [False, True])
def test_ties(gpu_lib, torch, halves):
    """angles of whole eighths and landings by powers of two: a half is common, and a result out of range"""
    case = many_rows(torch, 40, (4, 2, 64), halves=halves, deviation=3000.0)
    g = np.random.default_rng(40)
    rows = len(case["wide"])
    case["cos"], case["sin"] = ((g.integers(-12, 13, case["cos"].shape) << 27).astype(np.int32) for _ in range(2))
    case["cos"][0], case["sin"][0] = -(1 << 31), (1 << 31) - 1
    case["positions"][::50] = 0
    case["in_scales"][:, 0] = 1 << 30
    for name in ("k_landing", "v_landing"):
        case[name][:] = 1 << 30, -50 + 6, 1 << 32
    case["in_scales"][:, 1] = -50 + g.integers(-2, 3, rows)
    by_hundreds(gpu_lib, torch, case).compare(only=[0, 1, 50, 77, 299, 300, 600, rows - 1])


def test_values_at_the_ends(gpu_lib, torch):
    case = many_rows(torch, 41, (2, 1, 32))
    w = case["wide"]
    w[0], w[1], w[2], w[3], w[3, 5] = 0, -(1 << 31), (1 << 31) - 1, 0, 1
    w[4] = np.where(np.arange(128) % 2, 1 << 24, -(1 << 24) - 1)
    w[5], w[6] = 1 << 30, np.arange(128) - 64
    w[60:90] = np.random.default_rng(41).integers(-(1 << 31), 1 << 31, (30, 128))
    for r, (m, e) in {7: (1 << 30, 20), 8: ((1 << 31) - 1, -100), 9: (1 << 30, 60), 10: (1 << 30, 4096), 11: ((1 << 31) - 1, -4096), 61: (1 << 30, -60), 62: (1 << 30, -70)}.items():
        case["in_scales"][r] = m, e
    by_hundreds(gpu_lib, torch, case).compare(only=list(range(0, 13)) + list(range(58, 92)))


def test_some_refused_and_left_out(gpu_lib, torch):
    case = many_rows(torch, 42, (4, 2, 64))
    n, tables = len(case["wide"]), len(case["pages"])
    case["positions"][1] = -1
    case["positions"][2] = -2
    case["positions"][3] = 512
    case["places"][4] = 512
    case["places"][5] = -1
    case["table_of"][6] = tables
    case["table_of"][7] = -1
    case["pages"][tables - 1, case["places"][np.flatnonzero(case["table_of"] == tables - 1)[-1]] // PAGE] = -1
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
