"""ftb._runtime.zeroed_workspace, on CPU tensors with a fake of the stream."""
import contextlib

import pytest
import torch

from ftb import _lib, _runtime

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


def test_calls_whose_sizes_hardly_differ_share_a_buffer(stream):
    """More tokens take a few bytes more of plan; the parts that fill the workspace do not grow."""
    size = _lib.load().ftb_attention_workspace_bytes
    first = None
    for tokens in (300, 1000, 4093, 50000):
        ws = _runtime.zeroed_workspace(size(tokens, 8, tokens, 32, 8, 128), ZERO, CPU)
        first = ws if first is None else first
        assert ws is first, tokens
    assert first.numel() <= size(300, 8, 300, 32, 8, 128) * 9 // 8 and not _runtime._REPLACED


def test_small_sizes_are_not_rounded_to_large_ones(stream):
    for n in (1, 65536, 65537, 10 ** 6, 10 ** 7 + 1):
        _runtime._WS.clear()
        got = _runtime.zeroed_workspace(n, ZERO, CPU).numel()
        assert n <= got <= max(65536, n * 9 // 8 + 65536)
