"""The binding of the typed operators asks torch for the current device and stream by functions below its public ones; a torch without them serves as well."""
import types

import pytest


@pytest.fixture
def names():
    from dlprimitives_b200 import capi
    yield capi._Torch
    capi._Torch.load()                               # as it was, whatever a test took away


def test_without_the_inner_functions(names, monkeypatch):
    import torch
    for name in ("_cuda_getDevice", "_cuda_getCurrentRawStream"):
        monkeypatch.delattr(torch._C, name, raising=False)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 5)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device: types.SimpleNamespace(cuda_stream=1000 + device))
    names.load()
    assert names.current_device() == 5 and names.raw_stream(3) == 1003
    monkeypatch.undo()


def test_with_them(names, monkeypatch):
    import torch
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 2, raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda device: 77 + device, raising=False)
    names.load()
    assert names.current_device() == 2 and names.raw_stream(0) == 77
    monkeypatch.undo()


@pytest.mark.gpu
def test_a_call_through_the_public_functions(names, monkeypatch):
    import torch
    from dlprimitives_b200 import capi
    x, w = torch.randn(3, 64, device="cuda"), torch.ones(64, device="cuda")
    want, got = torch.empty_like(x), torch.zeros_like(x)
    capi.rms_norm(x, w, want)
    for name in ("_cuda_getDevice", "_cuda_getCurrentRawStream"):
        monkeypatch.delattr(torch._C, name, raising=False)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)               # (torch's own go through the names taken away)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device: types.SimpleNamespace(cuda_stream=0))
    names.load()
    capi.rms_norm(x, w, got)
    monkeypatch.undo()
    torch.cuda.synchronize()
    assert torch.equal(got, want)
