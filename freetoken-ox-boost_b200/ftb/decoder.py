"""A decoder layer around the MoE layer: norm -> qkv -> rotary positions and cache write -> paged
attention -> output projection -> gated residual and norm -> MoE -> gated residual and norm.

``AttnStep`` holds what one step of a batch needs on the device (built once per step, used by every
layer), ``PagedKvCache`` a layer's pages, ``DecoderLayer`` the weights. The projections are plain
matrix products (torch); everything between them is this package's kernels.
"""
from __future__ import annotations

from dataclasses import dataclass

import torch

from .attention import paged_attention
from .block import FP8, block_norm, rms_norm, rope_append


class PagedKvCache:
    """Keys and values of one layer in pages: ``k``, ``v`` [num_pages, page, kv heads, D]. With
    ``dtype=torch.float8_e4m3fn`` in 8 bits, with ``k_scale``, ``v_scale`` float32 [num_pages,
    page / scale_block, kv heads] (``scale_block`` tokens per scale: 16, 32, 64 or 128; by default the
    largest of them that divides the page)."""

    def __init__(self, num_pages: int, page: int, kv_heads: int, head_dim: int,
                 dtype=torch.bfloat16, device="cuda", scale_block: int | None = None):
        shape = (num_pages, page, kv_heads, head_dim)
        self.k = torch.zeros(shape, dtype=dtype, device=device)
        self.v = torch.zeros(shape, dtype=dtype, device=device)
        self.page = page
        self.k_scale = self.v_scale = None
        if dtype == FP8:
            size = scale_block
            if size is None:
                size = next((s for s in (128, 64, 32, 16) if page % s == 0), page)
            if size not in (16, 32, 64, 128) or page % size:
                raise ValueError(f"{size} tokens per scale in pages of {page}: expected 16, 32, 64 or "
                                 "128 that divide the page")
            # (0: no scale yet)
            self.k_scale, self.v_scale = (
                torch.zeros(num_pages, page // size, kv_heads, device=device) for _ in "kv")
        elif scale_block is not None:
            raise ValueError(f"scale_block={scale_block}: a cache of {dtype} has no scales")

    def tensors(self) -> list:
        """What a page id names, as :func:`~ftb.copy_pages` takes it."""
        return [self.k, self.v] + ([] if self.k_scale is None else [self.k_scale, self.v_scale])


@dataclass
class AttnStep:
    """The new tokens of a batch: rows of sequence b are ``cu_q[b]`` .. ``cu_q[b + 1]`` of the step's
    tokens (``cu_q`` None: one token each)."""
    positions: torch.Tensor    # int32 [tokens], or [axes, tokens]
    slots: torch.Tensor        # int32 [tokens]: page * page_size + row
    block_table: torch.Tensor  # int32 [batch, width]
    kv_len: torch.Tensor       # int32 [batch], with the new tokens
    cu_q: torch.Tensor | None
    max_q: int

    @classmethod
    def build(cls, pages: list, past: list, new: list, page: int, device="cuda",
              positions: torch.Tensor | None = None) -> "AttnStep":
        """From host lists: ``pages[b]`` the page ids of sequence b, ``past[b]`` the keys it has,
        ``new[b]`` its new tokens. ``positions`` replaces the running text positions."""
        if not len(pages) == len(past) == len(new):
            raise ValueError(f"{len(pages)} page lists, {len(past)} pasts, {len(new)} counts")
        at, slots, starts = [], [], [0]
        for ids, p, n in zip(pages, past, new):
            if p < 0 or n < 0 or p + n > len(ids) * page:
                raise ValueError(f"{p} + {n} keys do not fit {len(ids)} pages of {page}")
            at += range(p, p + n)
            slots += [ids[i // page] * page + i % page for i in range(p, p + n)]
            starts.append(starts[-1] + n)
        width = max([len(ids) for ids in pages] + [1])
        table = [list(ids) + [0] * (width - len(ids)) for ids in pages]

        def i32(x):
            return torch.tensor(x, dtype=torch.int32, device=device)

        most = max(new, default=0)
        decode = all(n == 1 for n in new)
        return cls(i32(at) if positions is None else positions, i32(slots),
                   i32(table).reshape(len(pages), width),
                   i32([p + n for p, n in zip(past, new)]), None if decode else i32(starts),
                   1 if decode else most)


class DecoderLayer:
    """Weights and forward pass of one layer. ``moe`` maps [tokens, H] to [tokens, H] (an
    ``Nvfp4MoELayer``). ``qkv`` [(q heads + 2 kv heads) * D, H], ``o`` [H, q heads * D]; norm
    weights [H]; the norms after the attention and after the MoE layer (``post_*``), the gates
    and the residual scale are optional."""

    def __init__(self, qkv: torch.Tensor, o: torch.Tensor, moe, input_norm: torch.Tensor,
                 moe_norm: torch.Tensor, q_heads: int, kv_heads: int, rope_table: torch.Tensor,
                 *, post_attn_norm=None, post_moe_norm=None, attn_gate=None, moe_gate=None,
                 residual_scale: float = 1.0, sections=None, order: str = "blocks",
                 pairs: str = "half", window: int = 0, eps: float = 1e-6):
        self.head_dim = o.shape[1] // q_heads
        if o.shape != (qkv.shape[1], q_heads * self.head_dim) or (
                qkv.shape[0] != (q_heads + 2 * kv_heads) * self.head_dim):
            raise ValueError(f"qkv {tuple(qkv.shape)} and o {tuple(o.shape)} do not fit {q_heads} "
                             f"query heads and {kv_heads} kv heads")
        self.qkv, self.o, self.moe = qkv, o, moe
        self.input_norm, self.moe_norm = input_norm, moe_norm
        self.post_attn_norm, self.post_moe_norm = post_attn_norm, post_moe_norm
        self.attn_gate, self.moe_gate = attn_gate, moe_gate
        self.residual_scale, self.eps, self.window = residual_scale, eps, window
        self.q_heads, self.kv_heads = q_heads, kv_heads
        self.rope_table = rope_table
        self.rope = dict(sections=sections, order=order, pairs=pairs)

    def attention(self, hidden: torch.Tensor, step: AttnStep, cache: PagedKvCache) -> torch.Tensor:
        """The attention block's output of normed ``hidden`` [tokens, H]; fills the cache."""
        qkv = (hidden @ self.qkv.t()).unflatten(1, (-1, self.head_dim))
        q, k, v = qkv.split([self.q_heads, self.kv_heads, self.kv_heads], 1)
        scales = {}
        if getattr(cache, "k_scale", None) is not None:
            scales = dict(k_scale=cache.k_scale, v_scale=cache.v_scale)
        q = rope_append(q, k, v, step.positions, self.rope_table, cache.k, cache.v, step.slots,
                        **scales, **self.rope)
        out = paged_attention(q, cache.k, cache.v, step.block_table, step.kv_len, step.cu_q,
                              step.max_q, window=self.window, **scales)
        return out.flatten(1) @ self.o.t()

    def forward(self, residual: torch.Tensor, hidden: torch.Tensor | None, step: AttnStep,
                cache: PagedKvCache, next_norm: torch.Tensor | None = None):
        """``(residual, hidden)`` after the layer. ``hidden`` is the residual stream through this
        layer's input norm (the last layer's second result; None: taken here), ``next_norm`` the
        weight of the norm that follows (the next layer's, or the model's last)."""
        if hidden is None:
            hidden = rms_norm(residual, self.input_norm, self.eps, out_dtype=self.qkv.dtype)
        y = self.attention(hidden, step, cache)
        residual, hidden = block_norm(residual, y, post_weight=self.post_attn_norm,
                                      gate=self.attn_gate, scale=self.residual_scale,
                                      pre_weight=self.moe_norm, eps=self.eps)
        y = self.moe(hidden)
        return block_norm(residual, y, post_weight=self.post_moe_norm, gate=self.moe_gate,
                          scale=self.residual_scale, pre_weight=next_norm, eps=self.eps)

    __call__ = forward
