"""Tensors on a GPU that is not the current one: a launch goes to the current device whatever its
pointers and its stream, so every entry point is called with the tensors' device made current.
With a fake of the devices and of the entry points: no kernel runs."""
import types

import pytest
import torch

from ftb import _lib, _runtime


class Devices:
    """The current device, torch.cuda.device, and entry points that note what was current."""

    def __init__(self, monkeypatch, current, status=0):
        self.current, self.seen, self.status = current, [], status
        outer = self

        class device:
            def __init__(self, d):
                self.to = d.index

            def __enter__(self):
                self.before, outer.current = outer.current, self.to

            def __exit__(self, *exc):
                outer.current = self.before

        monkeypatch.setattr(_runtime, "_current_device", lambda: self.current)
        monkeypatch.setattr(torch.cuda, "device", device)
        monkeypatch.setattr(_runtime, "stream_handle", lambda d: 1000 + d.index)
        monkeypatch.setattr(_lib, "load", lambda: types.SimpleNamespace(entry=self.entry))
        monkeypatch.setattr(_lib, "entry", lambda name: name)
        monkeypatch.setattr(_runtime, "_pycall", types.SimpleNamespace(call=self.call))

    def entry(self, *args):
        self.seen.append((self.current, args))
        return self.status

    def call(self, fn, args, pointers, stream, *tensors):
        self.seen.append((self.current, (fn, args, pointers, *tensors, stream)))
        return self.status


@pytest.mark.parametrize("current", [0, 1, 3])
def test_launches_run_on_the_tensors_device(monkeypatch, current):
    d = Devices(monkeypatch, current)
    _runtime.launch("entry", torch.device("cuda", 1), 7, 8)
    assert _runtime.caller(torch.device("cuda", 1))("name", b"args", (0,), 1001, "t") == 0
    assert d.seen == [(1, (7, 8, 1001)), (1, ("name", b"args", (0,), "t", 1001))]
    assert d.current == current


def test_the_device_comes_back_after_an_error(monkeypatch):
    d = Devices(monkeypatch, 0, status=_lib.FTB_ERR_SHAPE)
    monkeypatch.setattr(_lib, "status_string", lambda status: "shape")
    with pytest.raises(_lib.FtbError):
        _runtime.launch("entry", torch.device("cuda", 2), 7)
    assert _runtime.caller(torch.device("cuda", 2))("name", b"", (), 1002) == _lib.FTB_ERR_SHAPE
    assert [c for c, _ in d.seen] == [2, 2] and d.current == 0


@pytest.mark.parametrize("module", ["attention", "block", "ep", "fused_nvfp4", "fused_route"])
def test_every_launch_goes_this_way(module):
    """No module hands a stream to an entry point by itself (but a query of the group's own device)."""
    import importlib
    import inspect

    text = inspect.getsource(importlib.import_module(f"ftb.{module}"))
    left = [line for line in text.splitlines() if "stream_handle(" in line or "_pycall.call(" in line]
    assert all("caller(dev)" in line or "ftb_ep_status" in line for line in left), left
