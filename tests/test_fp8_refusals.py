"""Refusals of the 8-bit cache's calls that need no GPU: the C ABI's checks come before any launch, and
the Python entry points take CUDA tensors only."""
import ctypes

import pytest
import torch

import ftb
from ftb import _lib

OK, SHAPE, ALIGN, WORKSPACE, ARG = (_lib.FTB_OK, _lib.FTB_ERR_SHAPE, _lib.FTB_ERR_ALIGN,
                                    _lib.FTB_ERR_WORKSPACE, _lib.FTB_ERR_ARG)


def rope(**kw):
    a = dict(q=16, k=16, v=16, q_out=16, k_dst=16, v_dst=16, positions=16, table=16,
             table_rows=10, slots=16, n_slots=64, tokens=0, page=16, Hq=4, Hkv=2, D=64, rot=64,
             axes=1, sections=(32,))
    outer = dict(k_scale=16, v_scale=16, scale_block=16)
    for n in list(kw):
        if n in ("k_scale", "v_scale", "scale_block", "workspace", "workspace_bytes"):
            outer[n] = kw.pop(n)
    s = _lib.RopeFp8ArgsStruct(rope=_lib.RopeArgsStruct(**{**a, **kw}), **outer)
    return _lib.load().ftb_rope_fp8(ctypes.byref(s), None)


@pytest.mark.parametrize("kw,status", [
    (dict(), OK), (dict(tokens=-1), SHAPE), (dict(D=63), SHAPE), (dict(scale_block=8), SHAPE),
    (dict(scale_block=256, page=256), SHAPE), (dict(scale_block=32), SHAPE),
    (dict(scale_block=24, page=24), SHAPE), (dict(scale_block=32, page=48), SHAPE),
    (dict(type=2), ARG), (dict(tokens=4, slots=0), ARG), (dict(tokens=4, slots=0, v_dst=0), ARG),
    (dict(tokens=4, k_scale=0), ARG), (dict(tokens=4, v_scale=0), ARG), (dict(tokens=4, q=0), ARG),
    (dict(tokens=4, n_slots=63), SHAPE), (dict(tokens=4, n_slots=-16), SHAPE),
    (dict(tokens=2049), WORKSPACE), (dict(tokens=2049, workspace=16, workspace_bytes=65536), WORKSPACE),
    (dict(tokens=2049, workspace=18, workspace_bytes=1 << 20), ALIGN),
    (dict(tokens=4, Hkv=1025), SHAPE)])
def test_rope(kw, status):
    assert rope(**kw) == status


def test_rope_null():
    assert _lib.load().ftb_rope_fp8(None, None) == ARG


def test_rope_workspace_bytes():
    size = _lib.load().ftb_rope_fp8_workspace_bytes
    assert size(2048, 1 << 20) == _lib.FTB_ATTN_ZERO_BYTES
    assert size(2049, 1 << 20) == _lib.FTB_ATTN_ZERO_BYTES + (4 << 20)
    assert size(-1, 5) == 0


def attention(**kw):
    a = dict(q=256, k_cache=256, v_cache=256, block_table=256, kv_len=256, out=256, workspace=256,
             workspace_bytes=1 << 34, q_strides=(512, 128), k_strides=(8192, 256, 128),
             v_strides=(8192, 256, 128), total_q=4, num_pages=10, table_stride=8, batch=4, max_q=0,
             table_width=8, page=32, Hq=4, Hkv=2, D=128, causal=1, scale=0.1)
    outer = dict(k_scale=16, v_scale=16, scale_block=32)
    for n in list(kw):
        if n in outer:
            outer[n] = kw.pop(n)
    s = _lib.AttnFp8ArgsStruct(attn=_lib.AttnArgsStruct(**{**a, **kw}), **outer)
    return _lib.load().ftb_attention_fp8(ctypes.byref(s), None)


@pytest.mark.parametrize("kw,status", [
    (dict(), OK), (dict(scale_block=8), SHAPE), (dict(scale_block=64), SHAPE),
    (dict(scale_block=24), SHAPE), (dict(scale_block=256, page=256), SHAPE), (dict(D=72), SHAPE),
    (dict(D=8), SHAPE), (dict(D=144), SHAPE), (dict(page=8, scale_block=16), SHAPE),
    (dict(max_q=1, k_scale=0), ARG), (dict(max_q=1, v_scale=0), ARG), (dict(max_q=1, q=0), ARG),
    (dict(max_q=1, k_strides=(8192, 264, 128)), ALIGN), (dict(max_q=1, q=8), ALIGN),
    (dict(max_q=1, workspace=0), WORKSPACE), (dict(max_q=1, total_q=5), SHAPE)])
def test_attention(kw, status):
    assert attention(**kw) == status


def test_attention_null():
    assert _lib.load().ftb_attention_fp8(None, None) == ARG


def copy(n=0, num_pages=4, caches=(256,), strides=(64,), sizes=(64,), src=16, dst=16):
    s = _lib.PagesArgsStruct(n=n, num_pages=num_pages, n_caches=len(caches), src=src, dst=dst)
    for i, (c, st, b) in enumerate(zip(caches, strides, sizes)):
        s.caches[i], s.page_strides[i], s.page_bytes[i] = c, st, b
    return _lib.load().ftb_copy_pages(ctypes.byref(s), None)


@pytest.mark.parametrize("kw,status", [
    (dict(), OK), (dict(n=-1), SHAPE), (dict(num_pages=-1), SHAPE), (dict(n=3, num_pages=0), OK),
    (dict(n=3, caches=(), strides=(), sizes=()), OK), (dict(n=3, sizes=(0,)), OK),
    (dict(n=3, sizes=(-1,)), SHAPE), (dict(n=3, strides=(63,)), SHAPE), (dict(n=3, caches=(None,)), ARG),
    (dict(n=3, src=None), ARG), (dict(n=3, dst=None), ARG),
    (dict(n=1 << 40, sizes=(1 << 20,), strides=(1 << 20,)), SHAPE), (dict(n=1 << 50), SHAPE)])
def test_copy_pages(kw, status):
    assert copy(**kw) == status


def test_copy_pages_null():
    assert _lib.load().ftb_copy_pages(None, None) == ARG


def test_entry_points_take_cuda_tensors():
    q = torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    i = torch.zeros(4, dtype=torch.int32)
    cache = torch.zeros(2, 16, 2, 64, dtype=torch.uint8).view(torch.float8_e4m3fn)
    scale = torch.ones(2, 1, 2)
    table = ftb.rope_table(8, 64, device="cpu")
    for call in (lambda: ftb.rope_append(q, q, q, i, table, cache, cache, i, k_scale=scale, v_scale=scale),
                 lambda: ftb.paged_attention(q, cache, cache, i[:, None], i, k_scale=scale, v_scale=scale),
                 lambda: ftb.copy_pages([cache], [0], [1])):
        with pytest.raises(ValueError, match="CUDA"):
            call()


def test_scales_of_a_cache():
    """The checks of the scales, without a device."""
    from ftb.block import scale_block

    cpu = torch.device("cpu")
    cache = torch.zeros(2, 64, 3, 16)
    assert scale_block(cache, torch.ones(2, 4, 3), torch.ones(2, 4, 3), cpu) == 16
    assert scale_block(cache, torch.ones(2, 1, 3), torch.ones(2, 3, 1).transpose(1, 2), cpu) == 64
    good = torch.ones(2, 4, 3)
    for k, v in ((good, None), (None, good), (good, good[:, :2]), (good.double(), good.double()),
                 (torch.ones(2, 8, 3),) * 2, (torch.ones(2, 0, 3),) * 2, (torch.ones(2, 3, 3),) * 2,
                 (torch.ones(3, 4, 3),) * 2, (torch.ones(2, 4, 2),) * 2, (good[0], good[0])):
        with pytest.raises(ValueError):
            scale_block(cache, k, v, cpu)


def test_paged_cache():
    f8 = torch.float8_e4m3fn
    c = ftb.PagedKvCache(3, 64, 2, 128, dtype=f8, device="cpu", scale_block=32)
    assert c.k.dtype == f8 and c.k_scale.shape == (3, 2, 2) and len(c.tensors()) == 4
    assert ftb.PagedKvCache(3, 256, 2, 128, dtype=f8, device="cpu").k_scale.shape == (3, 2, 2)
    c = ftb.PagedKvCache(3, 64, 2, 128, device="cpu")
    assert c.k_scale is None and len(c.tensors()) == 2
    for bad in (dict(dtype=f8, scale_block=24), dict(dtype=f8, scale_block=128), dict(scale_block=32)):
        with pytest.raises(ValueError):
            ftb.PagedKvCache(3, 64, 2, 128, device="cpu", **bad)
    with pytest.raises(ValueError):
        ftb.PagedKvCache(3, 8, 2, 128, dtype=f8, device="cpu")
