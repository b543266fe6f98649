"""Attention of new tokens over a paged cache, on libftb (``ftb_attention`` in ``include/ftb.h``)."""
from __future__ import annotations

import torch

from . import _lib
from ._runtime import (_ARGS, _pycall, caller, read_status, remember, require_cuda, stream_handle,
                       zeroed_workspace)
from .block import _TYPE, FP8, scale_block

_POINTERS = _lib.offsets(_lib.AttnArgsStruct, "q", "k_cache", "v_cache", "block_table", "kv_len",
                         "cu_q", "out", "lse", "workspace")
# (the plain call's arguments are the first member)
_FP8_POINTERS = _POINTERS + _lib.offsets(_lib.AttnFp8ArgsStruct, "k_scale", "v_scale")


def _int32(t, name, shape, dev):
    if t.dtype != torch.int32 or t.device != dev or t.shape != shape or (
            not t.is_contiguous() and t.shape[-1] > 1 and t.stride(-1) != 1):
        raise ValueError(f"{name}: {tuple(t.shape)} {t.dtype} on {t.device}, expected int32 "
                         f"{shape} on {dev} with contiguous rows")


def _args(q, k_cache, v_cache, block_table, kv_len, cu_q, max_q, scale, causal, window,
          k_scale=None, v_scale=None):
    """The checks of a call, and its arguments without the pointers."""
    dev = require_cuda(q)
    fp8 = k_scale is not None or v_scale is not None
    cache_dtype = FP8 if fp8 else q.dtype
    if q.dim() != 3 or q.dtype not in _TYPE or q.stride(2) != 1:
        raise ValueError(f"q: {tuple(q.shape)} {q.dtype}, expected [total, heads, D] bf16 or f16 "
                         "with contiguous heads")
    total, Hq, D = q.shape
    for name, c in (("k_cache", k_cache), ("v_cache", v_cache)):
        if c.dim() != 4 or c.dtype != cache_dtype or c.device != dev or c.shape[3] != D or (
                c.stride(3) != 1) or c.shape != k_cache.shape:
            raise ValueError(f"{name}: {tuple(c.shape)} {c.dtype} on {c.device}, expected [pages, "
                             f"page, kv heads, {D}] {cache_dtype} with contiguous heads on {dev}")
    pages, page, Hkv, _ = k_cache.shape
    if Hkv < 1 or Hq % Hkv:
        raise ValueError(f"{Hq} query heads do not divide into {Hkv} kv heads")
    if block_table.dim() != 2:
        raise ValueError("block_table must be [batch, width]")
    batch, width = block_table.shape
    _int32(block_table, "block_table", (batch, width), dev)
    _int32(kv_len, "kv_len", (batch,), dev)
    if cu_q is not None:
        _int32(cu_q, "cu_q", (batch + 1,), dev)
    elif batch != total or max_q != 1:
        raise ValueError(f"without cu_q q has one row per sequence (got {total} rows, batch {batch}, "
                         f"max_q {max_q})")
    if window < 0 or max_q < 0:
        raise ValueError(f"window={window}, max_q={max_q}")
    # (bounds of any size: what lies past the rows and past every key says no more)
    max_q, window = min(max_q, total), min(window, 2 ** 31 - 1)
    nbytes = _lib.load().ftb_attention_workspace_bytes(total, batch, max_q, Hq, Hkv, D)
    a = _lib.AttnArgsStruct(
        workspace_bytes=nbytes, q_strides=q.stride()[:2], k_strides=k_cache.stride()[:3],
        v_strides=v_cache.stride()[:3], total_q=total, num_pages=pages,
        table_stride=block_table.stride(0), batch=batch, max_q=max_q, table_width=width,
        page=page, Hq=Hq, Hkv=Hkv, D=D, causal=int(causal), window=window,
        type=_TYPE[q.dtype], scale=D ** -0.5 if scale is None else scale)
    if not fp8:
        return a
    size = scale_block(k_cache, k_scale, v_scale, dev)
    return _lib.AttnFp8ArgsStruct(attn=a, k_scale_strides=k_scale.stride(),
                                  v_scale_strides=v_scale.stride(), scale_block=size)


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                    block_table: torch.Tensor, kv_len: torch.Tensor,
                    cu_q: torch.Tensor | None = None, max_q: int = 1, *,
                    scale: float | None = None, causal: bool = True, window: int = 0,
                    out: torch.Tensor | None = None, return_lse: bool = False,
                    check_status: bool = False, k_scale: torch.Tensor | None = None,
                    v_scale: torch.Tensor | None = None):
    """Attention of the new tokens of a batch over their sequences' pages; their own keys and
    values are in the caches already (``rope_append``).

    ``q`` [total, q heads, D]; caches [pages, page, kv heads, D] (any strides with contiguous
    heads); ``block_table`` int32 [batch, width]; ``kv_len`` int32 [batch], keys of each sequence
    with the new ones. ``cu_q`` int32 [batch + 1] gives the rows of each sequence in ``q`` and
    ``max_q`` the most of them; without ``cu_q`` every sequence has one new token (decode).
    Token i of n sees the keys up to its own position ``kv_len - n + i`` (``causal``), and no more
    than the last ``window`` of them (0: all). A token that sees none gets 0 (lse -inf).
    Returns out [total, q heads, D], with ``return_lse`` also the natural log of the sum of the
    exponentials, float32 [total, q heads]. ``check_status`` reads the stream's status word
    (synchronises) and raises on page ids, lengths or starts outside the tensors, of this call or of
    one before it that did not look. ``max_q`` and the table's width pick the kernel: pass no more
    than the batch needs where that is known on the host.

    With ``k_scale`` and ``v_scale``, float32 [pages, page / S, kv heads], the caches are
    ``torch.float8_e4m3fn`` as :func:`rope_append` fills them: an element stands for its number times
    the scale of its block of S tokens (16, 32, 64 or 128) and head. D is then a multiple of 16."""
    if type(max_q) is not int or type(window) is not int or type(causal) is not bool:
        max_q, window, causal = int(max_q), int(window), bool(causal)
    if scale is not None and type(scale) is not float:
        scale = float(scale)
    fp8 = k_scale is not None or v_scale is not None
    key = (_pycall.key(q, k_cache, v_cache, block_table, kv_len, cu_q, k_scale, v_scale) if fp8 else
           _pycall.key(q, k_cache, v_cache, block_table, kv_len, cu_q), max_q, scale, causal, window)
    known = _ARGS.get(key)
    if known is None:
        a = _args(q, k_cache, v_cache, block_table, kv_len, cu_q, max_q, scale, causal, window, k_scale,
                  v_scale)
        known = remember(key, a, a.attn.workspace_bytes if fp8 else a.workspace_bytes)
    dev = q.device
    if out is None:
        out = _pycall.empty(q, q)
    elif out.shape != q.shape or out.dtype != q.dtype or out.device != dev or not out.is_contiguous():
        raise ValueError("out must be contiguous, of q's shape and dtype")
    lse = q.new_empty(q.shape[:2], dtype=torch.float32) if return_lse else None
    ws = zeroed_workspace(known[1], _lib.FTB_ATTN_ZERO_BYTES, dev)
    if fp8:
        st = caller(dev)(_lib.entry("ftb_attention_fp8"), known[0], _FP8_POINTERS, stream_handle(dev), q,
                         k_cache, v_cache, block_table, kv_len, cu_q, out, lse, ws, k_scale, v_scale)
    else:
        st = caller(dev)(_lib.entry("ftb_attention"), known[0], _POINTERS, stream_handle(dev), q, k_cache,
                         v_cache, block_table, kv_len, cu_q, out, lse, ws)
    if st:
        _lib.check("ftb_attention_fp8" if fp8 else "ftb_attention", st)
    if check_status:
        status = read_status(ws)
        if status:
            ws[:4].zero_()
            raise ValueError(f"paged_attention: device status {status} (1: page id or kv_len "
                             "outside the cache, 2: cu_q outside q or above max_q, 4: timeout)")
    return (out, lse) if return_lse else out
