"""sslm_b200_fork_resident for a cache that has no sequences (any more): its pages may still be held, and are handed on."""
import ctypes as C

import numpy as np
import pytest

from superslm_b200 import abi

pytestmark = pytest.mark.gpu
OLD = -9


@pytest.fixture()
def torch():
    t = pytest.importorskip("torch")
    assert t.cuda.is_available()
    t.cuda.set_device(0)
    return t


def empty(torch, pages, width=3, planes=2):
    z = lambda *shape: torch.full(shape, OLD, dtype=torch.int32, device="cuda")      # noqa: E731
    held = torch.from_numpy(np.random.default_rng(pages).integers(0, 3, pages).astype(np.int32)).cuda()
    kv = torch.arange(planes * pages * 16, device="cuda").remainder(100).to(torch.int8).view(planes, pages, 16) if pages > 0 else None
    d = dict(kv=kv, holders=held, tables=z(0, width), lengths=z(0), parents=z(0))
    out = dict(out_holders=z(pages), out_tables=z(0, width), out_lengths=z(0), drawn=z(pages), moves=z(0, 2), counts=z(2), status=z(0))
    return d, out


@pytest.mark.parametrize("pages", [0, 1, 31, 700, 5000, 70001])
def test_holders_are_handed_on_and_nothing_is_counted(gpu_lib, torch, pages):
    d, out = empty(torch, pages)
    before = None if pages == 0 else d["kv"].clone()
    abi.Fork(gpu_lib, **d, **out).run()
    torch.cuda.synchronize()
    assert torch.equal(out["out_holders"], d["holders"]) and out["counts"].tolist() == [0, 0]
    assert (out["drawn"] == OLD).all() and (pages == 0 or torch.equal(d["kv"], before))


def test_captured_and_replayed(gpu_lib, torch):
    d, out = empty(torch, 300)
    call = abi.Fork(gpu_lib, **d, **out)
    call.run()
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        with torch.cuda.graph(graph, stream=stream):
            call.run()
    d["holders"].add_(1)
    out["counts"].fill_(OLD)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out["out_holders"], d["holders"]) and out["counts"].tolist() == [0, 0]


def test_the_outputs_it_needs(gpu_lib, torch):
    """holders may not be their own output; without counts there is nowhere to say how many"""
    d, out = empty(torch, 9)
    for change in (dict(out_holders=d["holders"].data_ptr()), dict(out_holders=None), dict(holders=None), dict(counts=None)):
        call = abi.Fork(gpu_lib, **d, **out)
        for k, v in change.items():
            setattr(call.args, k, v)
        assert gpu_lib.dll.sslm_b200_fork_resident(C.byref(call.args), None) == abi.ST["SSLM_INVALID_ARGUMENT"], change
    torch.cuda.synchronize()
    assert (out["out_holders"] == OLD).all() and (out["counts"] == OLD).all()
