"""Tensor checks, stream handles and per-stream workspaces for the libftb calls."""
from __future__ import annotations

import ctypes
import threading

import torch

from . import _lib

_pycall = _lib.Pycall()

_WS: dict = {}


# The current stream's handle without a Stream object around it (2.3 us less per call).
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def stream_handle(device: torch.device) -> int:
    if _raw_stream is not None and device.index is not None:
        return _raw_stream(device.index)
    return torch.cuda.current_stream(device).cuda_stream


_TURNS: dict = {}
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def launch(name: str, device: torch.device, *args) -> None:
    """Calls entry point ``name`` with ``args`` and ``device``'s current stream, and raises its
    errors. A launch goes to the current device, whatever its pointers: ``device`` is made that.
    Calls of one stream take turns between threads: one may be several launches over the stream's
    workspace, and the interpreter's lock is not held around them."""
    if _current_device() != device.index:
        with torch.cuda.device(device):
            return launch(name, device, *args)
    stream = stream_handle(device)
    key = (device.index, stream)
    with _TURNS.get(key) or _TURNS.setdefault(key, threading.Lock()):
        st = getattr(_lib.load(), name)(*args, stream)
    if st:
        _lib.check(name, st)


def caller(device: torch.device):
    """``_pycall.call``, with ``device`` current as in :func:`launch`."""
    if _current_device() == device.index:
        return _pycall.call

    def call(*args):
        with torch.cuda.device(device):
            return _pycall.call(*args)
    return call


def require_cuda(*tensors: torch.Tensor) -> torch.device:
    dev = tensors[0].device
    if dev.type != "cuda":
        raise ValueError(f"ftb ops run on CUDA tensors only (got {dev}); there is no CPU path")
    for t in tensors:
        if t.device != dev:
            raise ValueError(f"all tensors must be on {dev} (got {t.device})")
    return dev


def require(t: torch.Tensor, name: str, dtype=None, shape=None, contiguous=True) -> None:
    if dtype is not None and t.dtype != dtype:
        raise ValueError(f"{name}: dtype {t.dtype}, expected {dtype}")
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name}: shape {tuple(t.shape)}, expected {tuple(shape)}")
    if contiguous and not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


# Argument blocks of calls, all but their pointers, as they were when a call of that key was first
# checked: the checks cost more than the launch. A key holds what the checks look at: shape,
# strides, dtype and device of each tensor (_pycall.key, or the mark of a None in its place) and
# the options, as Python's own numbers: a tensor among them would be found again by its identity,
# whatever it holds by then.
_ARGS: dict = {}


def remember(key: tuple, args, *extra):
    """Keeps (and returns) the argument struct's bytes and what else the call needs to know."""
    if len(_ARGS) >= 4096:
        _ARGS.clear()
    known = _ARGS[key] = (bytes(args), *extra)
    return known


def workspace(nbytes: int, device: torch.device) -> torch.Tensor:
    """A cached uint8 device buffer of at least ``nbytes`` for the current stream.

    Grown (never shrunk) on demand; call once eagerly before CUDA-graph capture so capture
    does not allocate. Calls on one stream are ordered, so sharing it per stream is safe."""
    key = (device.index, stream_handle(device))
    t = _WS.get(key)
    if t is None or t.numel() < nbytes:
        t = torch.empty(max(int(nbytes), 1 << 16), dtype=torch.uint8, device=device)
        _WS[key] = t
    return t


_REPLACED: list = []


def zeroed_workspace(nbytes: int, zero_bytes: int, device: torch.device) -> torch.Tensor:
    """A cached buffer like :func:`workspace`, of its own, whose first ``zero_bytes`` are zero when
    it is made: for calls whose counters start at zero and are left at zero.

    A buffer that a larger one replaces stays allocated, since a captured graph may hold it (it
    grows by half at least: the old ones together are no more than twice the new one). Sizes are
    rounded up to an eighth of their power of two, so that calls whose sizes hardly differ share a
    buffer. One that is made under capture belongs to the graph alone: its counters are zeroed at
    each replay, not now."""
    key = (device.index, stream_handle(device), "zeroed")
    t = _WS.get(key)
    if t is None or t.numel() < nbytes:
        with torch.cuda.device(device):
            captured = torch.cuda.is_current_stream_capturing()
        if t is not None and not captured:
            _REPLACED.append(t)
            nbytes = max(nbytes, t.numel() * 3 // 2)
        step = 1 << max(16, int(nbytes).bit_length() - 4)
        nbytes = -(-int(nbytes) // step) * step
        t = torch.empty(nbytes, dtype=torch.uint8, device=device)
        t[:zero_bytes].zero_()
        if not captured:
            _WS[key] = t
    return t


def read_status(ws: torch.Tensor) -> int:
    """The device status word (first 4 bytes of a workspace); synchronises the stream."""
    return int(ws[:4].view(torch.int32).item())


def ptr(t: torch.Tensor | None):
    return None if t is None else ctypes.c_void_p(t.data_ptr())
