"""The stream that a prepared call runs on where its caller names none (no GPU is needed: torch and the verb are stood in for)."""
import contextlib
import types

import pytest

from superslm_b200 import abi

torch = pytest.importorskip("torch")


class Verb:
    def __call__(self, args, stream):
        self.stream = stream
        return 0


@pytest.fixture()
def call(monkeypatch):
    c = object.__new__(abi._ResidentCall)
    c._fn, c.verb, c.args, c._device = Verb(), "verb", abi.SampleArgs(), types.SimpleNamespace(index=3)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 3)
    monkeypatch.setattr(torch.cuda, "device", lambda d: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: types.SimpleNamespace(cuda_stream=70 + getattr(device, "index", device)))
    return c


def test_by_the_raw_handle_where_torch_gives_it(call, monkeypatch):
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 40 + index, raising=False)
    call.run()
    assert call._fn.stream == 43
    call.run(9)
    assert call._fn.stream == 9
    call.run(0)      # (the default stream, not "none named")
    assert call._fn.stream == 0


def test_by_the_public_call_where_it_does_not(call, monkeypatch):
    monkeypatch.delattr(torch._C, "_cuda_getCurrentRawStream", raising=False)
    call.run()
    assert call._fn.stream == 73
