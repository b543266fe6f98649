"""The append into an 8-bit cache writes each block's and head's scale: calls whose scales, or caches, share
their memory are refused before any launch (no GPU needed)."""
import ctypes

import pytest

from ftb import _lib

SHAPE, ARG = _lib.FTB_ERR_SHAPE, _lib.FTB_ERR_ARG


def rope(**kw):
    a = dict(q=16, k=16, v=16, q_out=16, k_dst=256, v_dst=512, positions=16, table=16, table_rows=10, slots=16,
             n_slots=64, tokens=4, page=32, Hq=4, Hkv=2, D=64, rot=64, axes=1, sections=(32,),
             k_dst_strides=(4096, 128, 64), v_dst_strides=(4096, 128, 64))
    outer = dict(k_scale=16, v_scale=32, k_scale_strides=(4, 2, 1), v_scale_strides=(4, 2, 1), scale_block=16)
    for n in list(kw):
        if n in outer:
            outer[n] = kw.pop(n)
    s = _lib.RopeFp8ArgsStruct(rope=_lib.RopeArgsStruct(**{**a, **kw}), **outer)
    return _lib.load().ftb_rope_fp8(ctypes.byref(s), None)


@pytest.mark.parametrize("kw,status", [
    (dict(v_scale=16), ARG), (dict(v_dst=256), ARG),
    *((dict([(n, (0, 2, 1))]), SHAPE) for n in ("k_scale_strides", "v_scale_strides")),
    *((dict([(n, (4, 0, 1))]), SHAPE) for n in ("k_scale_strides", "v_scale_strides")),
    *((dict([(n, (4, 2, 0))]), SHAPE) for n in ("k_scale_strides", "v_scale_strides")),
    *((dict([(n, (0, 128, 64))]), SHAPE) for n in ("k_dst_strides", "v_dst_strides")),
    *((dict([(n, (4096, 0, 64))]), SHAPE) for n in ("k_dst_strides", "v_dst_strides")),
    *((dict([(n, (4096, 128, 0))]), SHAPE) for n in ("k_dst_strides", "v_dst_strides"))])
def test_memory_of_its_own(kw, status):
    assert rope(**kw) == status
