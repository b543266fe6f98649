"""ftb._runtime.zeroed_workspace, on CPU tensors with a fake of the stream."""
import contextlib

import pytest
import torch

from ftb import _runtime

CPU = torch.device("cpu")
ZERO = 4096


@pytest.fixture
def stream(monkeypatch):
    """Capture state of the fake stream; allocations come filled with 0xff."""
    class Stream:
        capturing = False

    empty = torch.empty

    def filled(*size, **kw):
        return empty(*size, **kw).fill_(255)

    monkeypatch.setattr(_runtime, "_WS", {})
    monkeypatch.setattr(_runtime, "_REPLACED", [])
    monkeypatch.setattr(_runtime, "stream_handle", lambda device: 5)
    monkeypatch.setattr(torch.cuda, "device", lambda device: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: Stream.capturing)
    monkeypatch.setattr(torch, "empty", filled)
    return Stream


@pytest.mark.parametrize("capturing", [False, True])
def test_only_the_counters_are_zeroed(stream, capturing):
    """A workspace of a captured call is made in the graph, so what is zeroed is at each replay."""
    stream.capturing = capturing
    ws = _runtime.zeroed_workspace(1 << 20, ZERO, CPU)
    assert ws.numel() >= 1 << 20
    assert (ws[:ZERO] == 0).all() and (ws[ZERO:] == 255).all()


def test_a_captured_workspace_is_not_kept(stream):
    kept = _runtime.zeroed_workspace(10000, ZERO, CPU)
    stream.capturing = True
    assert _runtime.zeroed_workspace(10000, ZERO, CPU) is kept  # (made before the capture)
    larger = _runtime.zeroed_workspace(1 << 20, ZERO, CPU)
    stream.capturing = False
    assert _runtime.zeroed_workspace(10000, ZERO, CPU) is kept
    assert _runtime.zeroed_workspace(1 << 20, ZERO, CPU) is not larger
    assert any(t is kept for t in _runtime._REPLACED)
