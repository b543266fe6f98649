"""The operators of a decoder block around the MoE layer, on libftb: the norms before and after a
block with its gated residual, and the rotary positions with the write into the paged cache.

  * ``block_norm(x, y, ...)`` -> ``(r, h)``: r = x + scale * act(gate) * norm(y, post_weight),
    h = norm(r, pre_weight); ``rms_norm(x, weight)`` is its last step alone;
  * ``rope_table`` (cos and sin of every position), ``rope`` and ``rope_append``.

Shapes, types and strides are those of ``ftb_block_norm`` and ``ftb_rope`` in ``include/ftb.h``.
"""
from __future__ import annotations

import torch

from . import _lib
from ._runtime import (_ARGS, _pycall, caller, remember, require, require_cuda, stream_handle,
                       zeroed_workspace)

_TYPE = {torch.bfloat16: _lib.FTB_TYPE_BF16, torch.float16: _lib.FTB_TYPE_F16}
_GATE_ACTS = {None: _lib.FTB_GATE_LINEAR, "sigmoid": _lib.FTB_GATE_SIGMOID}
_PAIRS = {"half": _lib.FTB_PAIRS_HALF, "adjacent": _lib.FTB_PAIRS_ADJACENT}
_ORDERS = {"blocks": _lib.FTB_AXES_BLOCKS, "cyclic": _lib.FTB_AXES_CYCLIC}
_NORM_POINTERS = _lib.offsets(_lib.NormArgsStruct, "x", "y", "gate", "post", "pre", "r", "h")
_ROPE_POINTERS = _lib.offsets(_lib.RopeArgsStruct, "q", "k", "v", "q_out", "k_dst", "v_dst",
                              "positions", "table", "slots")
# (the plain call's arguments are the first member)
_ROPE_FP8_POINTERS = _ROPE_POINTERS + _lib.offsets(_lib.RopeFp8ArgsStruct, "k_scale", "v_scale",
                                                   "workspace")
FP8 = torch.float8_e4m3fn


def _row_stride(t: torch.Tensor, name: str) -> int:
    """The stride between rows of the last dimension; that dimension is contiguous."""
    if t.is_contiguous():
        return t.shape[-1]
    if t.dim() != 2 or (t.shape[1] > 1 and t.stride(1) != 1):
        raise ValueError(f"{name} must be contiguous, or 2-dimensional with contiguous rows")
    return t.stride(0)


def _new(like: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    if like.dtype == dtype:
        return _pycall.empty(like, like)
    return torch.empty(like.shape, dtype=dtype, device=like.device)


def _given(t: torch.Tensor, name: str, like: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    require(t, name, dtype, like.shape)
    if t.device != like.device:
        raise ValueError(f"{name} must be on {like.device}")
    return t


def _norm_args(x, y, gate, post, pre, scale, eps, gate_act, dtype):
    """The checks of a norm call, and its arguments without the pointers."""
    dev = require_cuda(x)
    H = x.shape[-1]
    a = _lib.NormArgsStruct()
    a.x_stride, a.H, a.rows = _row_stride(x, "x"), H, x.numel() // max(1, H)
    if dtype not in _TYPE:
        raise ValueError(f"{'x' if y is None else 'y'}: dtype {dtype}, expected bfloat16 or float16")
    if x.dtype not in (dtype, torch.float32):
        raise ValueError(f"x: dtype {x.dtype}, expected {dtype} or float32")
    if gate_act not in _GATE_ACTS:
        raise ValueError(f"gate_act={gate_act!r}: expected None or 'sigmoid'")
    a.type, a.gate_act = _TYPE[dtype], _GATE_ACTS[gate_act]
    a.residual_type = _lib.FTB_TYPE_F32 if x.dtype == torch.float32 else a.type
    a.scale, a.eps = scale, eps
    kind = None  # one dtype of gate and weights
    if post is not None:
        kind = _weight(post, "post_weight", H, dtype, dev, kind)
    if pre is not None:
        kind = _weight(pre, "pre_weight", H, dtype, dev, kind)
    if y is not None:
        if y.device != dev or y.shape != x.shape:
            raise ValueError(f"y: {tuple(y.shape)} on {y.device}, expected {tuple(x.shape)} on {dev}")
        a.y_stride = _row_stride(y, "y")
    if gate is not None:
        kind = _weight_dtype(gate, "gate", dtype, dev, kind)
        if gate.shape == x.shape and gate.dim() > 1:
            a.gate_kind, a.gate_stride = _lib.FTB_GATE_FULL, _row_stride(gate, "gate")
        elif gate.shape == (H,) and gate.is_contiguous():
            a.gate_kind = _lib.FTB_GATE_CHANNEL
        elif gate.shape == (*x.shape[:-1], 1):
            a.gate_kind = _lib.FTB_GATE_TOKEN
            a.gate_stride = 1 if gate.is_contiguous() or gate.dim() == 1 else _row_stride(gate, "gate")
        else:
            raise ValueError(f"gate: shape {tuple(gate.shape)}, expected contiguous [{H}], "
                             f"{(*x.shape[:-1], 1)} or {tuple(x.shape)}")
    a.weights_f32 = kind == torch.float32
    return a


def _launch_norm(args, x, y, gate, post, pre, r, h):
    dev = x.device
    st = caller(dev)(_lib.entry("ftb_block_norm"), args, _NORM_POINTERS, stream_handle(dev), x, y, gate,
                     post, pre, r, h)
    if st:
        _lib.check("ftb_block_norm", st)


def _weight_dtype(t, name, dtype, dev, kind):
    if t.device != dev or t.dtype not in (dtype, torch.float32) or (
            kind is not None and t.dtype != kind):
        raise ValueError(f"{name}: {t.dtype} on {t.device}, expected {dtype} or float32, the same "
                         f"for gate and weights, on {dev}")
    return t.dtype


def _weight(t, name, H, dtype, dev, kind):
    if t.shape != (H,) or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous [{H}] tensor, got {tuple(t.shape)}")
    return _weight_dtype(t, name, dtype, dev, kind)


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
    if y is None:
        raise ValueError("y is None: rms_norm(x, weight) is the norm alone")
    if type(scale) is not float or type(eps) is not float:
        scale, eps = float(scale), float(eps)
    key = (_pycall.key(x, y, gate, post_weight, pre_weight), scale, eps, gate_act)
    known = _ARGS.get(key) or remember(key, _norm_args(x, y, gate, post_weight, pre_weight, scale,
                                                       eps, gate_act, y.dtype))
    r = _pycall.empty(x, x) if residual_out is None else _given(residual_out, "residual_out", x, x.dtype)
    h = None
    if pre_weight is not None:
        h = _pycall.empty(x, y) if out is None else _given(out, "out", x, y.dtype)
    _launch_norm(known[0], x, y, gate, post_weight, pre_weight, r, h)
    return r, h


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6,
             out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """``x * rsqrt(mean(x^2) + eps) * weight`` over the last dimension, in ``out_dtype`` (``x``'s
    own, or bfloat16 for a float32 ``x``)."""
    dtype = out_dtype or (torch.bfloat16 if x.dtype == torch.float32 else x.dtype)
    if type(eps) is not float:
        eps = float(eps)
    key = (_pycall.key(x, weight), eps, dtype)
    known = _ARGS.get(key) or remember(key, _norm_args(x, None, None, None, weight, 1.0, eps, None,
                                                       dtype))
    h = _new(x, dtype)
    _launch_norm(known[0], x, None, None, None, weight, None, h)
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


def _heads(t, name, tokens, D, dtype, dev):
    """The (token, head) strides of [tokens, heads, D] with contiguous heads."""
    st = t.stride()
    if len(st) != 3 or st[2] != 1 or t.dtype != dtype or t.device != dev or t.shape[0] != tokens or (
            t.shape[2] != D):
        raise ValueError(f"{name}: {tuple(t.shape)} {t.dtype} strides {st} on {t.device}, "
                         f"expected [{tokens}, heads, {D}] {dtype} with contiguous heads on {dev}")
    return st[:2]


def _int_kind(t, name, dev):
    if t.dtype not in (torch.int32, torch.int64) or t.device != dev:
        raise ValueError(f"{name}: {t.dtype} on {t.device}, expected int32 or int64 on {dev}")
    return t.dtype == torch.int64


def scale_block(cache, k_scale, v_scale, dev) -> int:
    """The tokens per scale of an 8-bit cache [pages, page, kv heads, D], after the scales' checks."""
    pages, page, Hkv, _ = cache.shape
    for name, t in (("k_scale", k_scale), ("v_scale", v_scale)):
        if t is None:
            raise ValueError(f"{name} is None: an 8-bit cache has both scales")
        if t.dim() != 3 or t.dtype != torch.float32 or t.device != dev or t.shape != k_scale.shape or (
                t.shape[0] != pages or t.shape[2] != Hkv):
            raise ValueError(f"{name}: {tuple(t.shape)} {t.dtype} on {t.device}, expected float32 "
                             f"[{pages}, page / tokens per scale, {Hkv}] on {dev}")
    blocks = k_scale.shape[1]
    size = page // blocks if blocks else 0
    if size * blocks != page or size not in (16, 32, 64, 128):
        raise ValueError(f"{blocks} scales for a page of {page} tokens: expected 16, 32, 64 or 128 "
                         "tokens per scale")
    return size


def _rope_args(q, k, v, positions, table, k_dst, v_dst, slots, sections, order, pairs,
               cache_dtype=None):
    """The checks of a rotary call, and its arguments without the pointers."""
    dev = require_cuda(q)
    dtype = q.dtype
    if q.dim() != 3 or dtype not in _TYPE:
        raise ValueError(f"q: {tuple(q.shape)} {dtype}, expected [tokens, heads, D] bf16 or f16")
    tokens, Hq, D = q.shape
    a = _lib.RopeArgsStruct(q_strides=_heads(q, "q", tokens, D, dtype, dev),
                            k_strides=_heads(k, "k", tokens, D, dtype, dev), tokens=tokens,
                            Hq=Hq, Hkv=k.shape[1], D=D, type=_TYPE[dtype])
    Hkv = k.shape[1]
    if table.dim() != 2 or table.dtype != torch.float32 or not table.is_contiguous() or (
            table.device != dev):
        raise ValueError(f"table must be a contiguous float32 [positions, rot] on {dev}")
    a.table_rows, a.rot = table.shape
    if pairs not in _PAIRS or order not in _ORDERS:
        raise ValueError(f"pairs={pairs!r}, order={order!r}: expected one of {sorted(_PAIRS)}, "
                         f"{sorted(_ORDERS)}")
    a.pairs, a.order = _PAIRS[pairs], _ORDERS[order]
    a.pos64 = _int_kind(positions, "positions", dev)
    if positions.dim() not in (1, 2) or positions.shape[-1] != tokens or (
            tokens > 1 and positions.stride(-1) != 1):
        raise ValueError(f"positions: shape {tuple(positions.shape)}, expected [{tokens}] or "
                         f"[axes, {tokens}], contiguous along the tokens")
    a.axes = 1 if positions.dim() == 1 else positions.shape[0]
    a.pos_stride = positions.stride(0)
    half = table.shape[1] // 2
    sections = (half,) if sections is None else sections
    if len(sections) != a.axes or a.axes > 4 or sum(sections) != half or min(sections) < 0:
        raise ValueError(f"sections {sections}: expected {a.axes} counts (of at most 4 axes) that "
                         f"sum to {half}")
    a.sections = sections
    if slots is None:
        a.k_dst_strides = (0, Hkv * D, D)
        return a
    a.v_strides = _heads(v, "v", tokens, D, dtype, dev)
    cache_dtype = cache_dtype or dtype
    for name, c in (("k_cache", k_dst), ("v_cache", v_dst)):
        if c.dim() != 4 or c.shape != (*k_dst.shape[:2], Hkv, D) or c.dtype != cache_dtype or (
                c.device != dev or c.stride(3) != 1):
            raise ValueError(f"{name}: {tuple(c.shape)} {c.dtype} on {c.device}, expected [pages, "
                             f"page, {Hkv}, {D}] {cache_dtype} with contiguous heads on {dev}")
    if v.shape[1] != Hkv:
        raise ValueError(f"v: shape {tuple(v.shape)}, expected {tuple(k.shape)}")
    a.slot64 = _int_kind(slots, "slots", dev)
    if slots.shape != (tokens,) or not slots.is_contiguous():
        raise ValueError(f"slots must be a contiguous [{tokens}] tensor")
    a.k_dst_strides, a.v_dst_strides = k_dst.stride()[:3], v_dst.stride()[:3]
    a.page = k_dst.shape[1]
    a.n_slots = k_dst.shape[0] * k_dst.shape[1]
    return a


def _rope(q, k, v, positions, table, k_dst, v_dst, slots, sections, order, pairs, q_out):
    if sections is not None:
        sections = tuple(map(int, sections))
    key = (_pycall.key(q, k, positions, table) if slots is None else
           _pycall.key(q, k, positions, table, v, k_dst, v_dst, slots), sections, order, pairs)
    known = _ARGS.get(key) or remember(key, _rope_args(q, k, v, positions, table, k_dst, v_dst, slots,
                                                       sections, order, pairs))
    out = _pycall.empty(q, q) if q_out is None else _given(q_out, "q_out", q, q.dtype)
    if q.shape[0]:
        dev = q.device
        st = caller(dev)(_lib.entry("ftb_rope"), known[0], _ROPE_POINTERS, stream_handle(dev), q, k, v,
                         out, k_dst, v_dst, positions, table, slots)
        if st:
            _lib.check("ftb_rope", st)
    return out


def _rope_fp8(q, k, v, positions, table, k_cache, v_cache, slots, sections, order, pairs, q_out,
              k_scale, v_scale):
    """The call into an 8-bit cache."""
    if slots is None or v is None:
        raise ValueError("an 8-bit cache takes v and the slots of the tokens")
    if sections is not None:
        sections = tuple(map(int, sections))
    key = (_pycall.key(q, k, positions, table, v, k_cache, v_cache, slots, k_scale, v_scale), sections,
           order, pairs)
    known = _ARGS.get(key)
    if known is None:
        a = _rope_args(q, k, v, positions, table, k_cache, v_cache, slots, sections, order, pairs, FP8)
        size = scale_block(k_cache, k_scale, v_scale, q.device)
        nbytes = _lib.load().ftb_rope_fp8_workspace_bytes(a.tokens, a.n_slots)
        b = _lib.RopeFp8ArgsStruct(rope=a, k_scale_strides=k_scale.stride(),
                                   v_scale_strides=v_scale.stride(), workspace_bytes=nbytes,
                                   scale_block=size)
        known = remember(key, b, nbytes if nbytes > _lib.FTB_ATTN_ZERO_BYTES else 0)
    out = _pycall.empty(q, q) if q_out is None else _given(q_out, "q_out", q, q.dtype)
    if q.shape[0]:
        dev = q.device
        ws = zeroed_workspace(known[1], _lib.FTB_ATTN_ZERO_BYTES, dev) if known[1] else None
        st = caller(dev)(_lib.entry("ftb_rope_fp8"), known[0], _ROPE_FP8_POINTERS, stream_handle(dev), q,
                         k, v, out, k_cache, v_cache, positions, table, slots, k_scale, v_scale, ws)
        if st:
            _lib.check("ftb_rope_fp8", st)
    return out


def rope(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, table: torch.Tensor, *,
         sections=None, order: str = "blocks", pairs: str = "half"):
    """``(q, k)`` [tokens, heads, D] turned by their positions [tokens] or [axes, tokens]; the
    other arguments are those of :func:`rope_append`."""
    k_out = torch.empty(k.shape, dtype=k.dtype, device=k.device)
    return _rope(q, k, None, positions, table, k_out, None, None, sections, order, pairs,
                 None), k_out


def rope_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor,
                table: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                slots: torch.Tensor, *, sections=None, order: str = "blocks",
                pairs: str = "half", q_out: torch.Tensor | None = None,
                k_scale: torch.Tensor | None = None,
                v_scale: torch.Tensor | None = None) -> torch.Tensor:
    """Turns q and k by their positions, writes the turned k and v into the caches [pages, page,
    kv heads, D] and returns the turned q (in ``q_out``, which may be a contiguous ``q``).

    ``slots`` [tokens]: page * page_size + row of each token, -1 for one that is not stored.
    ``positions`` [tokens], or [axes, tokens] with ``sections``, the number of frequencies of each
    axis: in ``order="blocks"`` one axis after another, in ``"cyclic"`` the axes in turn.
    ``pairs="half"`` turns (x[i], x[i + rot/2]), ``"adjacent"`` (x[2i], x[2i+1]), for the first
    rot = table.shape[1] elements of a head; the rest is copied.

    With ``k_scale`` and ``v_scale``, float32 [pages, page / S, kv heads], the caches are
    ``torch.float8_e4m3fn``, and an element stands for its number times the scale of its block of S
    tokens (16, 32, 64 or 128) and head. Scales are powers of two; that of a block is set by the largest
    element when its first row is written, and grows with what joins the block, whose older rows are
    then rounded again (``ftb_rope_fp8`` in ``include/ftb.h`` has the rule)."""
    if k_scale is not None or v_scale is not None:
        return _rope_fp8(q, k, v, positions, table, k_cache, v_cache, slots, sections, order, pairs,
                         q_out, k_scale, v_scale)
    return _rope(q, k, v, positions, table, k_cache, v_cache, slots, sections, order, pairs, q_out)
