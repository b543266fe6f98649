"""Entry points called from several threads: a call may be several launches over its stream's
workspace, so calls of one stream must not interleave. Those of different streams may: a launch can
wait for its stream, and that for a peer whose stream another thread has to feed."""
import ctypes
import threading
import time
import types

import torch

from ftb import _lib, _pycall, _runtime


def overlaps(streams):
    """How often a call of a stream began while another of the same stream was under way."""
    inside, found = {}, []

    @ctypes.CFUNCTYPE(ctypes.c_int, ctypes.c_void_p, ctypes.c_void_p)
    def entry(args, stream):
        inside[stream] = inside.get(stream, 0) + 1
        found.append(inside[stream] > 1)
        time.sleep(0.005)  # (lets other threads in)
        inside[stream] -= 1
        return 0

    fn = ctypes.cast(entry, ctypes.c_void_p).value
    start = threading.Barrier(len(streams))

    def work(stream):
        start.wait()
        for _ in range(8):
            assert _pycall.call(fn, bytes(8), (), stream) == 0

    threads = [threading.Thread(target=work, args=(s,)) for s in streams]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
        assert not t.is_alive()
    assert len(found) == 8 * len(streams)
    return sum(found)


def test_calls_of_one_stream_take_turns():
    assert overlaps([64] * 4) == 0
    assert overlaps([64, 64, 4096, 4096]) == 0


def test_a_waiting_call_holds_up_its_own_stream_only():
    free = threading.Event()

    @ctypes.CFUNCTYPE(ctypes.c_int, ctypes.c_void_p, ctypes.c_void_p)
    def entry(args, stream):
        return 0 if stream != 16 or free.wait(60) else 1

    fn = ctypes.cast(entry, ctypes.c_void_p).value
    first = threading.Thread(target=lambda: _pycall.call(fn, bytes(8), (), 16))
    first.start()
    for stream in range(32, 32 + 16 * 200, 16):
        assert _pycall.call(fn, bytes(8), (), stream) == 0
    free.set()
    first.join(60)
    assert not first.is_alive()


def test_launch_takes_turns_too(monkeypatch):
    """_runtime.launch, the way of the entry points without an argument struct."""
    current, inside, found = threading.local(), {}, []

    def entry(arg, stream):
        inside[stream] = inside.get(stream, 0) + 1
        found.append(inside[stream] > 1)
        time.sleep(0.005)
        inside[stream] -= 1
        return 0

    monkeypatch.setattr(_runtime, "_current_device", lambda: 0)
    monkeypatch.setattr(_runtime, "stream_handle", lambda d: current.stream)
    monkeypatch.setattr(_lib, "load", lambda: types.SimpleNamespace(entry=entry))

    def work(stream):
        current.stream = stream
        for _ in range(8):
            _runtime.launch("entry", torch.device("cuda", 0), 1)

    threads = [threading.Thread(target=work, args=(s,)) for s in (64, 64, 64, 4096)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    assert len(found) == 32 and sum(found) == 0
