"""ftb._pycall: the signature of a call's tensors, and the call of a C entry point (here a Python
callback with the entry points' C signature)."""
import ctypes

import pytest
import torch

import ftb  # noqa: F401
from ftb import _lib, _pycall


def test_key_holds_shape_strides_dtype_and_device():
    a = torch.zeros(4, 6, dtype=torch.bfloat16)
    same = _pycall.key(torch.ones(4, 6, dtype=torch.bfloat16))
    assert _pycall.key(a) == same  # (not the address)
    others = [a.half(), a.t(), a[:, :3], a[:3], a.view(2, 2, 6), a.view(24), a.to("meta"),
              torch.zeros(8, 6, dtype=torch.bfloat16)[::2]]
    keys = [same] + [_pycall.key(t) for t in others]
    assert len(set(keys)) == len(keys)


def test_key_of_several_arguments():
    a, b, s = torch.zeros(3), torch.zeros(3, 3), torch.zeros(())
    made = [_pycall.key(*x) for x in ((a,), (a, None), (None, a), (a, b), (b, a), (s, a), (None,), ())]
    assert len(set(made)) == len(made)


def test_key_refuses():
    with pytest.raises(TypeError):
        _pycall.key([1, 2])
    with pytest.raises(ValueError):
        _pycall.key(*[torch.zeros(2, 2, 2)] * 60)


class Args(ctypes.Structure):
    _fields_ = [("n", ctypes.c_int64), ("x", ctypes.c_void_p), ("y", ctypes.c_void_p)]


def test_call_writes_the_pointers():
    seen = []

    @ctypes.CFUNCTYPE(ctypes.c_int, ctypes.POINTER(Args), ctypes.c_void_p)
    def entry(args, stream):
        seen.append((args.contents.n, args.contents.x, args.contents.y, stream))
        return 3

    fn = ctypes.cast(entry, ctypes.c_void_p).value
    at = _lib.offsets(Args, "x", "y")
    template = bytes(Args(n=7))
    t = torch.zeros(5)
    assert _pycall.call(fn, template, at, 64, t[2:], None) == 3
    assert seen == [(7, t.data_ptr() + 8, None, 64)]
    assert template == bytes(Args(n=7))
    for bad in ((fn, template, at, 0, t), (fn, template, (20, 8), 0, t, t), (0, template, at, 0, t, t),
                (fn, template, at, 0, t, 5), (fn, b"x" * 2000, at, 0, t, t), (fn, "no", at, 0, t, t)):
        with pytest.raises((TypeError, ValueError)):
            _pycall.call(*bad)
    assert len(seen) == 1


def test_empty():
    a = torch.zeros(4, 8, 6).half()[:, 1:5]
    e = _pycall.empty(a, torch.zeros(1, dtype=torch.bfloat16))
    assert e.shape == a.shape and e.is_contiguous() and e.dtype == torch.bfloat16
    with pytest.raises(TypeError):
        _pycall.empty(a)
