"""The operators of a decoder block around the MoE layer, on libftb: the norms before and after a
block with its gated residual, and the rotary positions with the write into the paged cache.

  * ``block_norm(x, y, ...)`` -> ``(r, h)``: r = x + scale * act(gate) * norm(y, post_weight),
    h = norm(r, pre_weight); ``rms_norm(x, weight)`` is its last step alone;
  * ``rope_table`` (cos and sin of every position), ``rope`` and ``rope_append``.

Shapes, types and strides are those of ``ftb_block_norm`` and ``ftb_rope`` in ``include/ftb.h``.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from ._runtime import require, require_cuda, stream_handle

_TYPE = {torch.bfloat16: _lib.FTB_TYPE_BF16, torch.float16: _lib.FTB_TYPE_F16}
_GATE_ACTS = {None: _lib.FTB_GATE_LINEAR, "sigmoid": _lib.FTB_GATE_SIGMOID}
_PAIRS = {"half": _lib.FTB_PAIRS_HALF, "adjacent": _lib.FTB_PAIRS_ADJACENT}
_ORDERS = {"blocks": _lib.FTB_AXES_BLOCKS, "cyclic": _lib.FTB_AXES_CYCLIC}


def _rows(t: torch.Tensor, name: str):
    """``t`` as rows of its last dimension: (rows, row stride)."""
    if t.dim() == 1:
        return 1, t.shape[0]
    if t.dim() == 2:
        if t.shape[1] > 1 and t.stride(1) != 1:
            raise ValueError(f"{name}: the last dimension must be contiguous")
        return t.shape[0], t.stride(0)
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous or 2-dimensional")
    return t.numel() // max(1, t.shape[-1]), t.shape[-1]


def _weight(t, name, H, act_dtype, dev):
    if t is None:
        return 0, None
    if t.dtype not in (act_dtype, torch.float32):
        raise ValueError(f"{name}: dtype {t.dtype}, expected {act_dtype} or float32")
    if t.shape != (H,) or not t.is_contiguous() or t.device != dev:
        raise ValueError(f"{name} must be a contiguous [{H}] tensor on {dev}")
    return t.data_ptr(), t.dtype


def _launch_norm(x, y, gate, post, pre, scale, eps, gate_act, dtype, r, h):
    dev = require_cuda(x)
    H = x.shape[-1]
    rows, x_stride = _rows(x, "x")
    a = _lib.NormArgsStruct(rows=rows, x=x.data_ptr(), x_stride=x_stride, H=H, type=_TYPE[dtype],
                            residual_type=_lib.FTB_TYPE_F32 if x.dtype == torch.float32
                            else _TYPE[dtype], scale=scale, eps=eps)
    kinds = set()
    for name, t in (("post_weight", post), ("pre_weight", pre)):
        p, kind = _weight(t, name, H, dtype, dev)
        setattr(a, "post" if t is post and name == "post_weight" else "pre", p)
        kinds.add(kind)
    if y is not None:
        if y.device != dev or y.shape != x.shape:
            raise ValueError(f"y: {tuple(y.shape)} on {y.device}, expected {tuple(x.shape)} on {dev}")
        a.y = y.data_ptr()
        a.y_stride = _rows(y, "y")[1]
    if gate is not None:
        if gate.device != dev or gate.dtype not in (dtype, torch.float32):
            raise ValueError(f"gate: {gate.dtype} on {gate.device}, expected {dtype} or float32 on {dev}")
        kinds.add(gate.dtype)
        if gate.shape == (H,) and (x.dim() > 1 or H != rows):
            a.gate_kind = _lib.FTB_GATE_CHANNEL
            if not gate.is_contiguous():
                raise ValueError("gate must be contiguous")
        elif gate.shape == x.shape:
            a.gate_kind = _lib.FTB_GATE_FULL
            a.gate_stride = _rows(gate, "gate")[1]
        elif gate.shape == (*x.shape[:-1], 1):
            a.gate_kind = _lib.FTB_GATE_TOKEN
            a.gate_stride = _rows(gate, "gate")[1]
        else:
            raise ValueError(f"gate: shape {tuple(gate.shape)}, expected [{H}], "
                             f"{(*x.shape[:-1], 1)} or {tuple(x.shape)}")
        a.gate = gate.data_ptr()
        a.gate_act = gate_act
    kinds.discard(None)
    if len(kinds) > 1:
        raise ValueError("gate, post_weight and pre_weight must have one dtype")
    a.weights_f32 = int(torch.float32 in kinds)
    if r is not None:
        a.r = r.data_ptr()
    if h is not None:
        a.h = h.data_ptr()
    st = _lib.load().ftb_block_norm(ctypes.byref(a), stream_handle(dev))
    _lib.check("ftb_block_norm", st)


def _out(t, name, like, dtype):
    if t is None:
        return torch.empty(like.shape, dtype=dtype, device=like.device)
    require(t, name, dtype, like.shape)
    if t.device != like.device:
        raise ValueError(f"{name} must be on {like.device}")
    return t


def block_norm(x: torch.Tensor, y: torch.Tensor, *, post_weight: torch.Tensor | None = None,
               gate: torch.Tensor | None = None, scale: float = 1.0,
               pre_weight: torch.Tensor | None = None, eps: float = 1e-6, gate_act=None,
               residual_out: torch.Tensor | None = None, out: torch.Tensor | None = None):
    """``(r, h)`` of a block's output ``y`` (bf16 or f16, [..., H]) and the residual stream ``x``
    (the same type, or float32)::

        r = x + scale * act(gate) * (rms(y) * post_weight  or  y)
        h = rms(r) * pre_weight                              (None without pre_weight)

    ``gate``: [H], [..., 1] or [..., H], through a sigmoid with ``gate_act="sigmoid"``.
    ``residual_out`` may be ``x`` and ``out`` may be ``y``."""
    if y.dtype not in _TYPE:
        raise ValueError(f"y: dtype {y.dtype}, expected bfloat16 or float16")
    if x.dtype not in (y.dtype, torch.float32):
        raise ValueError(f"x: dtype {x.dtype}, expected {y.dtype} or float32")
    if gate_act not in _GATE_ACTS:
        raise ValueError(f"gate_act={gate_act!r}: expected None or 'sigmoid'")
    require_cuda(x)
    r = _out(residual_out, "residual_out", x, x.dtype)
    h = _out(out, "out", x, y.dtype) if pre_weight is not None else None
    _launch_norm(x, y, gate, post_weight, pre_weight, float(scale), float(eps),
                 _GATE_ACTS[gate_act], y.dtype, r, h)
    return r, h


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6,
             out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """``x * rsqrt(mean(x^2) + eps) * weight`` over the last dimension, in ``out_dtype`` (``x``'s
    own, or bfloat16 for a float32 ``x``)."""
    dtype = out_dtype or (torch.bfloat16 if x.dtype == torch.float32 else x.dtype)
    if dtype not in _TYPE or x.dtype not in (dtype, torch.float32):
        raise ValueError(f"rms_norm from {x.dtype} to {dtype}")
    require_cuda(x)
    h = torch.empty(x.shape, dtype=dtype, device=x.device)
    _launch_norm(x, None, None, None, weight, 1.0, float(eps), 0, dtype, None, h)
    return h


def rope_table(positions: int, rot: int, theta: float = 10000.0, device="cuda",
               inv_freq: torch.Tensor | None = None) -> torch.Tensor:
    """[positions, rot] float32: cos and then sin of p * theta^(-2i/rot) (or p * inv_freq[i]),
    computed in 64 bits: in 32 the angle of a late position is off by more than bf16 resolves."""
    if inv_freq is None:
        inv_freq = float(theta) ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    w = inv_freq.to(device=device, dtype=torch.float64)
    if w.shape != (rot // 2,):
        raise ValueError(f"inv_freq: shape {tuple(w.shape)}, expected ({rot // 2},)")
    angle = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * w
    return torch.cat([angle.cos(), angle.sin()], 1).float()


def _heads(t, name, tokens, dtype, dev, D=None):
    if t.dim() != 3 or t.shape[0] != tokens or t.dtype != dtype or t.device != dev or (
            D is not None and t.shape[2] != D) or t.stride(2) != 1:
        raise ValueError(f"{name}: {tuple(t.shape)} {t.dtype} strides {t.stride()} on {t.device}, "
                         f"expected [{tokens}, heads, {D or 'D'}] {dtype} with contiguous heads on {dev}")


def _int_kind(t, name, dev):
    if t.dtype not in (torch.int32, torch.int64) or t.device != dev:
        raise ValueError(f"{name}: {t.dtype} on {t.device}, expected int32 or int64 on {dev}")
    return int(t.dtype == torch.int64)


def _rope(q, k, v, positions, table, sections, order, pairs, q_out, a):
    dev = require_cuda(q)
    if q.dim() != 3 or q.dtype not in _TYPE:
        raise ValueError(f"q: {tuple(q.shape)} {q.dtype}, expected [tokens, heads, D] bf16 or f16")
    tokens, Hq, D = q.shape
    _heads(q, "q", tokens, q.dtype, dev)
    _heads(k, "k", tokens, q.dtype, dev, D)
    if table.dim() != 2 or table.dtype != torch.float32 or not table.is_contiguous() or table.device != dev:
        raise ValueError(f"table must be a contiguous float32 [positions, rot] on {dev}")
    rot = table.shape[1]
    if pairs not in _PAIRS or order not in _ORDERS:
        raise ValueError(f"pairs={pairs!r}, order={order!r}: expected one of {sorted(_PAIRS)}, "
                         f"{sorted(_ORDERS)}")
    a.pos64 = _int_kind(positions, "positions", dev)
    axes = 1 if positions.dim() == 1 else positions.shape[0]
    if positions.dim() not in (1, 2) or positions.shape[-1] != tokens or (
            tokens > 1 and positions.stride(-1) != 1):
        raise ValueError(f"positions: shape {tuple(positions.shape)}, expected [{tokens}] or "
                         f"[axes, {tokens}], contiguous along the tokens")
    sections = (rot // 2,) if sections is None else tuple(int(n) for n in sections)
    if len(sections) != axes or axes > 4 or sum(sections) != rot // 2 or min(sections) < 0:
        raise ValueError(f"sections {sections}: expected {axes} counts (of at most 4 axes) that "
                         f"sum to {rot // 2}")
    out = _out(q_out, "q_out", q, q.dtype)
    a.q, a.k, a.q_out = q.data_ptr(), k.data_ptr(), out.data_ptr()
    a.q_strides[:] = q.stride()[:2]
    a.k_strides[:] = k.stride()[:2]
    a.positions, a.table, a.table_rows = positions.data_ptr(), table.data_ptr(), table.shape[0]
    a.pos_stride = positions.stride(0) if positions.dim() == 2 else 0
    a.tokens, a.Hq, a.Hkv, a.D, a.rot = tokens, Hq, k.shape[1], D, rot
    a.axes, a.order, a.pairs, a.type = axes, _ORDERS[order], _PAIRS[pairs], _TYPE[q.dtype]
    for i, n in enumerate(sections):
        a.sections[i] = n
    if tokens:
        st = _lib.load().ftb_rope(ctypes.byref(a), stream_handle(dev))
        _lib.check("ftb_rope", st)
    return out


def rope(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, table: torch.Tensor, *,
         sections=None, order: str = "blocks", pairs: str = "half"):
    """``(q, k)`` [tokens, heads, D] turned by their positions [tokens] or [axes, tokens]."""
    a = _lib.RopeArgsStruct()
    k_out = torch.empty(k.shape, dtype=k.dtype, device=k.device)
    a.k_dst = k_out.data_ptr()
    if k.dim() == 3:
        a.k_dst_strides[:] = (0, k_out.stride(0), k_out.stride(1))
    return _rope(q, k, None, positions, table, sections, order, pairs, None, a), k_out


def rope_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor,
                table: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                slots: torch.Tensor, *, sections=None, order: str = "blocks",
                pairs: str = "half", q_out: torch.Tensor | None = None) -> torch.Tensor:
    """Turns q and k by their positions, writes the turned k and v into the caches [pages, page,
    kv heads, D] and returns the turned q.

    ``slots`` [tokens]: page * page_size + row of each token, -1 for one that is not stored.
    ``positions`` [tokens], or [axes, tokens] with ``sections``, the number of frequencies of each
    axis: in ``order="blocks"`` one axis after another, in ``"cyclic"`` the axes in turn.
    ``pairs="half"`` turns (x[i], x[i + rot/2]), ``"adjacent"`` (x[2i], x[2i+1]), for the first
    rot = table.shape[1] elements of a head; the rest is copied."""
    a = _lib.RopeArgsStruct()
    dev = require_cuda(q)
    _heads(k, "k", k.shape[0], q.dtype, dev)
    _heads(v, "v", k.shape[0], q.dtype, dev, k.shape[2])
    want = (k_cache.shape[0], k_cache.shape[1] if k_cache.dim() == 4 else 0, k.shape[1], k.shape[2])
    for name, c in (("k_cache", k_cache), ("v_cache", v_cache)):
        if c.dtype != q.dtype or c.device != dev or tuple(c.shape) != want or c.stride(3) != 1:
            raise ValueError(f"{name}: {tuple(c.shape)} {c.dtype} on {c.device}, expected [pages, "
                             f"page, {k.shape[1]}, {k.shape[2]}] {q.dtype} with contiguous rows on {dev}")
    if v.shape != k.shape:
        raise ValueError(f"v: shape {tuple(v.shape)}, expected {tuple(k.shape)}")
    if slots.shape != (k.shape[0],) or not slots.is_contiguous():
        raise ValueError(f"slots must be a contiguous [{k.shape[0]}] tensor")
    a.slot64 = _int_kind(slots, "slots", dev)
    a.v, a.k_dst, a.v_dst, a.slots = v.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), slots.data_ptr()
    a.v_strides[:] = v.stride()[:2]
    a.k_dst_strides[:] = k_cache.stride()[:3]
    a.v_dst_strides[:] = v_cache.stride()[:3]
    a.page = k_cache.shape[1]
    a.n_slots = k_cache.shape[0] * k_cache.shape[1]
    return _rope(q, k, v, positions, table, sections, order, pairs, q_out, a)
