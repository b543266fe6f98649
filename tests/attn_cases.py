"""Paged-attention cases for the tests: inputs with every unused cache row poisoned, and the
definition in 64 bits with the error bound of each output element.

Bound of an output o = sum p_j v_j (p the softmax) against 64 bits, elementwise, with u the unit
roundoff of the tensors' type (2^-8 bf16, 2^-11 f16) and A = sum p_j |v_j|:
  u |o|     the output's rounding
  u A       each p_j is rounded to the type as the tensor cores' operand
  2^-13 A   fp32 scores (|s| <= 2^4, 2^-22 relative each way, exponentiated) and an exponential
            that is exact to 2^-14
  f16 only: a p_j below 2^-14 of the row's reference is subnormal, 2^-25 absolute each:
            2^-25 sum |v_j| / l, with l >= 2^-8 of the sum where the reference is at most 2^8
            above the row's maximum (a lazily moved maximum), so 2^-17 sum |v_j| / l_max
lse: 2^-14 + 2^-21 |lse|.
"""
import math
from dataclasses import dataclass, field

import torch

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


@dataclass
class AttnCase:
    pairs: list  # (new tokens, keys) of each sequence
    q_heads: int = 8
    kv_heads: int = 2
    head: int = 128
    page: int = 16
    dtype: torch.dtype = torch.bfloat16
    window: int = 0
    causal: bool = True
    scale: float | None = None
    layout: str = "nhd"  # or "hnd": heads before the rows of a page
    q_slice: bool = False  # q is a slice of a wider row (fused projection)
    cu: bool = True  # pass cu_q
    poison: float = math.nan
    seed: int = 0
    spread: float = 1.0  # standard deviation of q: larger makes the softmax sharper
    t: dict = field(default_factory=dict)


def build(c: AttnCase, device="cuda"):
    g = torch.Generator().manual_seed(c.seed)
    total = sum(n for n, _ in c.pairs)
    used = sum(-(-kv // c.page) for _, kv in c.pairs)
    pages = used + 3
    order = torch.randperm(pages, generator=g)
    width = max(1, max((-(-kv // c.page) for _, kv in c.pairs), default=1)) + 1
    table = torch.full((len(c.pairs), width), -7, dtype=torch.int32)  # unused entries: no page
    q = (torch.randn(total, c.q_heads, c.head, generator=g) * c.spread).to(c.dtype)
    caches = []
    keys = [torch.randn(kv, 2, c.kv_heads, c.head, generator=g).to(c.dtype) for _, kv in c.pairs]
    for which in range(2):
        cache = torch.full((pages, c.page, c.kv_heads, c.head), c.poison, dtype=c.dtype)
        at = 0
        for b, (n, kv) in enumerate(c.pairs):
            count = -(-kv // c.page)
            ids = order[at:at + count]
            at += count
            table[b, :count] = ids.int()
            flat = torch.full((count * c.page, c.kv_heads, c.head), c.poison, dtype=c.dtype)
            flat[:kv] = keys[b][:, which]
            if c.window:  # rows below every token's window were given up
                flat[:max(0, kv - n - c.window + 1)] = c.poison
            cache[ids] = flat.view(count, c.page, c.kv_heads, c.head)
        if c.layout == "hnd":
            cache = cache.transpose(1, 2).contiguous().to(device).transpose(1, 2)
        else:
            cache = cache.to(device)
        caches.append(cache)
    if c.q_slice:
        wide = torch.full((total, c.q_heads + 2, c.head), math.nan, dtype=c.dtype)
        wide[:, 1:-1] = q
        qd = wide.to(device)[:, 1:-1]
    else:
        qd = q.to(device)
    starts = [0]
    for n, _ in c.pairs:
        starts.append(starts[-1] + n)
    c.t = dict(q=qd, k_cache=caches[0], v_cache=caches[1], block_table=table.to(device),
               kv_len=torch.tensor([kv for _, kv in c.pairs], dtype=torch.int32, device=device),
               cu_q=torch.tensor(starts, dtype=torch.int32, device=device) if c.cu else None,
               max_q=max([n for n, _ in c.pairs] + [1]))
    return q, keys


def reference(c: AttnCase, q, keys):
    """(out, bound, lse) in 64 bits."""
    G = c.q_heads // c.kv_heads
    scale = c.head ** -0.5 if c.scale is None else c.scale
    out = torch.zeros(q.shape, dtype=torch.float64)
    bound = torch.zeros(q.shape, dtype=torch.float64)
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64)
    u = U[c.dtype]
    at = 0
    for (n, kv), x in zip(c.pairs, keys):
        rows = slice(at, at + n)
        at += n
        if n == 0 or kv == 0:
            continue
        place = torch.arange(kv - n, kv)[:, None]
        j = torch.arange(kv)
        seen = torch.ones(n, kv, dtype=torch.bool)
        if c.causal:
            seen &= j <= place
        if c.window:
            seen &= j > place - c.window
        k, v = x[:, 0].double(), x[:, 1].double()
        k, v = (y.repeat_interleave(G, 1).transpose(0, 1) for y in (k, v))  # [heads, kv, D]
        s = torch.matmul(q[rows].double().transpose(0, 1), k.transpose(1, 2)) * scale
        s = s.masked_fill(~seen, -math.inf)
        top = s.amax(-1, keepdim=True).clamp_min(-1e300)
        p = (s - top).exp()
        l = p.sum(-1, keepdim=True)
        live = l > 0
        w = torch.where(live, p / torch.where(live, l, 1.0), 0.0)
        o, a = w @ v, w @ v.abs()
        e = u * (o.abs() + a) + 2.0 ** -13 * a
        if c.dtype == torch.float16:
            e = e + 2.0 ** -17 * (seen.double() @ v.abs()) / torch.where(live, l, 1.0)
            e = e + 2.0 ** -25  # the output's own subnormals
        out[rows], bound[rows] = o.transpose(0, 1), e.transpose(0, 1)
        lse[rows] = torch.where(live, top + l.log(), -math.inf).squeeze(-1).transpose(0, 1)
    return out, bound * 1.01 + 1e-30, lse
