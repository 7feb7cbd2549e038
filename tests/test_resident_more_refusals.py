"""What the q/k/v site, the draw, forks and compaction refuse before they launch anything (no GPU is needed: no address is read)."""
import ctypes as C

import pytest

from superslm_b200 import abi, build

BAD, OFF, AT = abi.ST["SSLM_INVALID_ARGUMENT"], abi.ST["SSLM_MISALIGNED_BUFFER"], 1 << 20


@pytest.fixture(scope="module")
def dll():
    import os
    return C.CDLL(build.LIB if os.path.exists(build.LIB) else build.build())


def made(kind, base, change):
    a = kind(struct_size=C.sizeof(kind), **base)
    for k, v in change.items():
        setattr(a, k, v)
    return a


def site(**change):
    return made(abi.QkvSiteArgs, dict(rows=4, heads=12, kv_heads=2, head_dim=128, rotary=128, num_positions=100, num_tables=4, table_pages=7, q_shift=0, k_shift=0, q=AT, k=AT, v=AT,
                                      q_stride=2048, k_stride=2048, v_stride=2048, in_scales=AT, positions=AT, places=AT, table_of=AT, pages=AT, pages_stride=7, cos=AT, sin=AT,
                                      q_site_m=1 << 30, q_site_e=-30, k_landing=AT, v_landing=AT, khead=AT, kv=AT, num_pages=50, q_codes=AT, q_codes_stride=1536, q_scales=AT, consts=AT,
                                      saturations=AT, row_status=AT), change)


def sample(**change):
    return made(abi.SampleArgs, dict(rows=4, vocab=100, logits=AT, logits_stride=100, params=AT, draws=AT, out_tokens=AT, out_mass=AT, out_kept=AT, row_status=AT), change)


PAGES = dict(sequences=4, table_pages=7, planes=3, page_bytes=512, num_pages=50, kv=AT, holders=AT, tables=AT, tables_stride=7, lengths=AT, out_holders=2 * AT, out_tables=2 * AT,
             out_stride=7, moves=AT, counts=AT, status=AT)


def fork(**change):
    return made(abi.ForkArgs, dict(PAGES, parents=AT, grow=AT, out_lengths=2 * AT, drawn=AT), change)


def compact(**change):
    return made(abi.CompactArgs, dict(PAGES, new_of=AT), change)


@pytest.mark.parametrize("change,want", [
    (dict(struct_size=8), BAD), (dict(rows=-1), BAD), (dict(heads=-1), BAD), (dict(kv_heads=0), BAD), (dict(head_dim=96), BAD), (dict(heads=254, q_stride=1 << 16, q_codes_stride=1 << 16), BAD),
    (dict(heads=1 << 30), BAD), (dict(rotary=4), BAD), (dict(rotary=136), BAD), (dict(rotary=-8), BAD), (dict(halves=2), BAD), (dict(num_positions=-1), BAD), (dict(q_stride=1532), BAD),
    (dict(k_stride=252), BAD), (dict(v_stride=252), BAD), (dict(q_codes_stride=1532), BAD), (dict(q_gain=AT), BAD), (dict(k_gain=AT, k_shift=63), BAD), (dict(num_tables=-1), BAD),
    (dict(table_pages=-1), BAD), (dict(pages_stride=6), BAD), (dict(num_pages=-1), BAD), (dict(num_pages=1 << 31), BAD), (dict(q_site_m=1 << 31), BAD), (dict(q_site_m=5), BAD),
    (dict(q_site_e=5000), BAD), (dict(q=None, k=None, v=None), BAD), (dict(heads=0, k=None, v=None), BAD), (dict(k=None), BAD), (dict(v=None), BAD), (dict(positions=None), BAD), (dict(cos=None), BAD),
    (dict(sin=None), BAD), (dict(q_codes=None), BAD), (dict(khead=None), BAD), (dict(kv=None), BAD), (dict(pages=None), BAD), (dict(k_landing=None), BAD), (dict(v_landing=None), BAD),
    (dict(in_scales=None), BAD), (dict(table_of=None, num_tables=3), BAD), (dict(reserved=1), BAD),
    (dict(q=AT + 4), OFF), (dict(k=AT + 8), OFF), (dict(v=AT + 4), OFF), (dict(cos=AT + 4), OFF), (dict(kv=AT + 8), OFF), (dict(q_stride=2049), OFF), (dict(q_codes_stride=1538), OFF),
    (dict(q_codes=AT + 2), OFF), (dict(positions=AT + 2), OFF), (dict(in_scales=AT + 4), OFF), (dict(consts=AT + 4), OFF), (dict(k_landing=AT + 4), OFF)])
def test_site(dll, change, want):
    assert dll.sslm_b200_qkv_site_resident(C.byref(site(**change)), None) == want


@pytest.mark.parametrize("change,want", [
    (dict(struct_size=8), BAD), (dict(rows=-1), BAD), (dict(rows=65536), BAD), (dict(vocab=0), BAD), (dict(vocab=(1 << 20) + 1, logits_stride=1 << 21), BAD), (dict(logits_stride=99), BAD),
    (dict(logits=None), BAD), (dict(params=None), BAD), (dict(draws=None), BAD), (dict(out_tokens=None, out_mass=None, out_kept=None), BAD), (dict(reserved=1), BAD),
    (dict(logits=AT + 2), OFF), (dict(params=AT + 2), OFF), (dict(draws=AT + 1), OFF), (dict(out_mass=AT + 4), OFF), (dict(out_kept=AT + 2), OFF), (dict(row_status=AT + 2), OFF)])
def test_sample(dll, change, want):
    assert dll.sslm_b200_sample_resident(C.byref(sample(**change)), None) == want


BOTH = [(dict(struct_size=8), BAD), (dict(sequences=-1), BAD), (dict(sequences=65536), BAD), (dict(table_pages=-1), BAD), (dict(table_pages=65537, tables_stride=1 << 17, out_stride=1 << 17), BAD),
        (dict(num_pages=-1), BAD), (dict(num_pages=1 << 31), BAD), (dict(planes=-1), BAD), (dict(page_bytes=0), BAD), (dict(page_bytes=24), BAD), (dict(tables_stride=6), BAD), (dict(out_stride=6), BAD),
        (dict(reserved=1), BAD), (dict(holders=None), BAD), (dict(tables=None), BAD), (dict(lengths=None), BAD), (dict(out_holders=None), BAD), (dict(out_tables=None), BAD), (dict(moves=None), BAD),
        (dict(counts=None), BAD), (dict(out_holders=AT), BAD), (dict(moves=AT + 4), OFF), (dict(kv=AT + 8), OFF), (dict(tables=AT + 2), OFF), (dict(holders=AT + 1), OFF), (dict(status=AT + 2), OFF)]


@pytest.mark.parametrize("change,want", BOTH + [(dict(parents=None), BAD), (dict(out_lengths=None), BAD), (dict(status=None), BAD), (dict(drawn=None), BAD), (dict(out_tables=AT), BAD),
                                                (dict(out_lengths=AT), BAD), (dict(parents=AT + 2), OFF), (dict(grow=AT + 2), OFF)])
def test_fork(dll, change, want):
    assert dll.sslm_b200_fork_resident(C.byref(fork(**change)), None) == want


@pytest.mark.parametrize("change,want", BOTH + [(dict(new_of=None), BAD), (dict(new_of=AT + 2), OFF)])
def test_compact(dll, change, want):
    assert dll.sslm_b200_compact_resident(C.byref(compact(**change)), None) == want


def test_no_call_and_nothing_to_do(dll):
    for name in ("qkv_site", "sample", "fork", "compact"):
        assert getattr(dll, "sslm_b200_%s_resident" % name)(None, None) == BAD
    none = {k: None for k in ("q", "k", "v", "in_scales", "positions", "places", "table_of", "q_codes", "q_scales", "consts", "saturations", "row_status")}
    assert dll.sslm_b200_qkv_site_resident(C.byref(site(rows=0, **none)), None) == 0
    none = {k: None for k in ("logits", "params", "draws", "out_tokens", "out_mass", "out_kept", "row_status")}
    assert dll.sslm_b200_sample_resident(C.byref(sample(rows=0, **none)), None) == 0
    none = {k: None for k in ("tables", "lengths", "parents", "grow", "out_tables", "out_lengths", "moves", "status")}
    assert dll.sslm_b200_fork_resident(C.byref(fork(sequences=0, **none)), None) == 0


def test_prepared_calls_check_their_tensors():
    torch = pytest.importorskip("torch")
    lib = abi.SslmLib(build.LIB)
    z = lambda *shape, dtype=torch.int32: torch.zeros(shape, dtype=dtype)      # noqa: E731
    with pytest.raises(ValueError, match="GPU"):
        abi.Sample(lib, z(2, 8), z(2, 5), z(2), out_tokens=z(2))
    with pytest.raises(TypeError, match="logits"):
        abi.Sample(lib, z(2, 8, dtype=torch.float32), z(2, 5), z(2), out_tokens=z(2))
    with pytest.raises(ValueError, match="kv"):
        abi.Compact(lib, z(3, 4, 16, dtype=torch.int8), z(5), z(1, 2), z(1), z(5), z(1, 2), z(5), z(2, 2), z(2))
    with pytest.raises(ValueError, match="q, or k and v"):
        abi.QkvSite(lib, None, None, None, None, z(2), z(4, 8), z(4, 8))
