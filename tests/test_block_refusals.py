"""The block operators' refusals that need no GPU: the C ABI's checks come before any launch, and
the Python entry points take CUDA tensors only."""
import ctypes

import pytest
import torch

import ftb
from ftb import _lib

OK, SHAPE, ALIGN, WORKSPACE, ARG = (_lib.FTB_OK, _lib.FTB_ERR_SHAPE, _lib.FTB_ERR_ALIGN,
                                    _lib.FTB_ERR_WORKSPACE, _lib.FTB_ERR_ARG)


def norm(**kw):
    a = dict(x=16, y=16, r=16, h=16, pre=16, rows=4, x_stride=64, y_stride=64, H=64, eps=1e-6)
    s = _lib.NormArgsStruct(**{**a, **kw})
    return _lib.load().ftb_block_norm(ctypes.byref(s), None)


@pytest.mark.parametrize("kw,status", [
    (dict(H=0), SHAPE), (dict(H=16385), SHAPE), (dict(rows=-1), SHAPE), (dict(rows=0), OK),
    (dict(type=2), ARG), (dict(type=0, residual_type=1), ARG), (dict(gate_kind=4), ARG),
    (dict(gate_act=2), ARG), (dict(x=0), ARG), (dict(r=0), ARG), (dict(h=0), ARG),
    (dict(gate_kind=1), ARG), (dict(gate=16), ARG), (dict(y=0), ARG), (dict(y=0, r=0, pre=0), ARG)])
def test_norm(kw, status):
    assert norm(**kw) == status


def rope(**kw):
    a = dict(q=16, k=16, v=16, q_out=16, k_dst=16, v_dst=16, positions=16, table=16,
             table_rows=10, slots=16, n_slots=64, tokens=4, page=16, Hq=4, Hkv=2, D=64, rot=64,
             axes=1, sections=(32,))
    s = _lib.RopeArgsStruct(**{**a, **kw})
    return _lib.load().ftb_rope(ctypes.byref(s), None)


@pytest.mark.parametrize("kw,status", [
    (dict(tokens=0), OK), (dict(tokens=-1), SHAPE), (dict(D=63), SHAPE), (dict(D=514), SHAPE),
    (dict(rot=66, sections=(33,)), SHAPE), (dict(rot=31), SHAPE), (dict(axes=0), SHAPE),
    (dict(axes=5), SHAPE), (dict(sections=(31,)), SHAPE), (dict(axes=2, sections=(33, -1)), SHAPE),
    (dict(D=512, rot=258, sections=(129,)), SHAPE), (dict(table_rows=0), SHAPE),
    (dict(type=2), ARG), (dict(pairs=2), ARG), (dict(order=2), ARG), (dict(q=0), ARG),
    (dict(table=0), ARG), (dict(v_dst=0), ARG), (dict(page=0), ARG), (dict(slots=0), ARG)])
def test_rope(kw, status):
    assert rope(**kw) == status


def attention(**kw):
    a = dict(q=256, k_cache=256, v_cache=256, block_table=256, kv_len=256, out=256, workspace=256,
             workspace_bytes=1 << 34, q_strides=(512, 128), k_strides=(8192, 256, 128),
             v_strides=(8192, 256, 128), total_q=4, num_pages=10, table_stride=8, batch=4, max_q=1,
             table_width=8, page=32, Hq=4, Hkv=2, D=128, causal=1, scale=0.1)
    s = _lib.AttnArgsStruct(**{**a, **kw})
    return _lib.load().ftb_attention(ctypes.byref(s), None)


@pytest.mark.parametrize("kw,status", [
    (dict(batch=0), OK), (dict(max_q=0), OK), (dict(total_q=0), OK), (dict(total_q=-1), SHAPE),
    (dict(Hq=3), SHAPE), (dict(Hq=0), SHAPE), (dict(Hq=258), SHAPE), (dict(D=136), SHAPE),
    (dict(D=12), SHAPE), (dict(page=24), SHAPE), (dict(page=4), SHAPE), (dict(num_pages=0), SHAPE),
    (dict(window=-1), SHAPE), (dict(total_q=5), SHAPE), (dict(table_width=1 << 27), SHAPE),
    (dict(type=2), ARG), (dict(q=0), ARG), (dict(kv_len=0), ARG), (dict(out=0), ARG),
    (dict(scale=float("inf")), ARG), (dict(scale=float("nan")), ARG), (dict(q=8), ALIGN),
    (dict(k_strides=(8192, 250, 128)), ALIGN), (dict(q_strides=(512, 4)), ALIGN),
    (dict(workspace=0), WORKSPACE), (dict(workspace_bytes=100), WORKSPACE),
    (dict(workspace=128), ALIGN)])
def test_attention(kw, status):
    assert attention(**kw) == status


def test_attention_workspace_bytes():
    size = _lib.load().ftb_attention_workspace_bytes
    assert size(4, 4, 1, 32, 8, 128) > _lib.FTB_ATTN_ZERO_BYTES
    assert size(4096, 1, 4096, 32, 8, 128) > size(64, 64, 1, 32, 8, 128)
    assert size(4, 4, 1, 7, 0, 128) == 0


def test_entry_points_take_cuda_tensors():
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    q = torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    i = torch.zeros(4, dtype=torch.int32)
    cache = torch.zeros(2, 16, 2, 64, dtype=torch.bfloat16)
    table = ftb.rope_table(8, 64, device="cpu")
    for call in (lambda: ftb.block_norm(x, x), lambda: ftb.rms_norm(x, x[0]),
                 lambda: ftb.rope(q, q, i, table),
                 lambda: ftb.rope_append(q, q, q, i, table, cache, cache, i),
                 lambda: ftb.paged_attention(q, cache, cache, i[:, None], i)):
        with pytest.raises(ValueError, match="CUDA"):
            call()


def test_attn_step():
    step = ftb.AttnStep.build([[3, 1], [0]], [15, 0], [3, 2], 16, device="cpu")
    assert step.positions.tolist() == [15, 16, 17, 0, 1]
    assert step.slots.tolist() == [3 * 16 + 15, 16, 17, 0, 1]
    assert step.kv_len.tolist() == [18, 2] and step.cu_q.tolist() == [0, 3, 5]
    assert step.block_table.tolist() == [[3, 1], [0, 0]] and step.max_q == 3
    step = ftb.AttnStep.build([[3, 1], [0]], [15, 0], [1, 1], 16, device="cpu")
    assert step.cu_q is None and step.max_q == 1
    for bad in (([[0]], [16], [1]), ([[0]], [-1], [1]), ([[0]], [0], [0, 1])):
        with pytest.raises(ValueError):
            ftb.AttnStep.build(*bad, 16, device="cpu")
