"""The stream of a call without a `stream` argument, with and without torch's short way."""
import types

import pytest

import lucciola as L

torch = pytest.importorskip("torch")


@pytest.fixture(autouse=True)
def fresh(monkeypatch):
    monkeypatch.setattr(L, "_raw_stream", None, raising=False)
    monkeypatch.setattr(torch.cuda, "init", lambda: None)
    monkeypatch.setattr(torch.cuda, "current_stream",
                        lambda: types.SimpleNamespace(cuda_stream=1234))


def test_a_given_stream():
    assert L._stream(types.SimpleNamespace(cuda_stream=77)) == 77


def test_the_short_way_takes_the_current_device(monkeypatch):
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 3, raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda d: 500 + d, raising=False)
    assert L._stream() == 503
    assert L._stream() == 503


@pytest.mark.parametrize("name", ["_cuda_getDevice", "_cuda_getCurrentRawStream"])
def test_a_torch_without_it(monkeypatch, name):
    monkeypatch.delattr(torch._C, name, raising=False)
    assert L._stream() == 1234
    assert L._stream() == 1234
