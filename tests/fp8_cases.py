"""Cases of the 8-bit cache for the tests: inputs whose unused rows and scales hold NaN, and the
definitions in 64 bits.

Attention, bound of an output o = sum p_j v_j (p the softmax, v_j = c_j vs_j, a code times its block's
scale) against 64 bits, elementwise, with u the unit roundoff of the outputs' type and A = sum p_j |v_j|:
  u |o|       the output's rounding
  2^-11 A     each weight p_j vs_j / max is rounded to f16 as the tensor cores' operand (codes are exact)
  2^-13 A     fp32 scores (|s| <= 2^4, with log2 vs_j below 2^6) and an exponential exact to 2^-14
  2^-25 max_j(p_j vs_j) sum |c_j|   weights that are subnormal in f16, relative to the largest
  2^-25       f16 only: the output's own subnormals
lse: 2^-14 + 2^-21 |lse|.

Append: the rule in 32 bits, whose products and sums are single operations here as there: codes and
scales are equal, bit for bit.
"""
import math
from dataclasses import dataclass, field

import torch

from tests.attn_cases import U

FP8 = torch.float8_e4m3fn
NAN_CODE = 0x7f


@dataclass
class Fp8Case:
    pairs: list  # (new tokens, keys) of each sequence
    q_heads: int = 8
    kv_heads: int = 2
    head: int = 128
    page: int = 16
    block: int = 16
    dtype: torch.dtype = torch.bfloat16
    window: int = 0
    causal: bool = True
    scale: float | None = None
    layout: str = "nhd"  # or "hnd": heads before the rows of a page
    q_slice: bool = False  # q is a slice of a wider row (fused projection)
    cu: bool = True  # pass cu_q
    seed: int = 0
    spread: float = 1.0  # standard deviation of q
    steps: tuple = (-8, -5)  # log2 of the scales
    odd_scales: bool = False  # scales that are no powers of two
    t: dict = field(default_factory=dict)


def build(c: Fp8Case, device="cuda"):
    """Fills c.t with the call's arguments; (q, per sequence the codes and scales of each key) on the
    CPU."""
    g = torch.Generator().manual_seed(c.seed)
    total = sum(n for n, _ in c.pairs)
    used = sum(-(-kv // c.page) for _, kv in c.pairs)
    pages = used + 3
    order = torch.randperm(pages, generator=g)
    width = max(1, max((-(-kv // c.page) for _, kv in c.pairs), default=1)) + 1
    table = torch.full((len(c.pairs), width), -7, dtype=torch.int32)  # unused entries: no page
    q = (torch.randn(total, c.q_heads, c.head, generator=g) * c.spread).to(c.dtype)
    per_page = c.page // c.block
    tensors, keys = {}, [[] for _ in c.pairs]
    for name in "kv":
        codes = torch.full((pages, c.page, c.kv_heads, c.head), NAN_CODE, dtype=torch.uint8)
        scales = torch.full((pages, per_page, c.kv_heads), math.nan)
        at = 0
        for b, (n, kv) in enumerate(c.pairs):
            count = -(-kv // c.page)
            ids = order[at:at + count]
            at += count
            table[b, :count] = ids.int()
            flat = torch.full((count * c.page, c.kv_heads, c.head), NAN_CODE, dtype=torch.uint8)
            x = (torch.randn(kv, c.kv_heads, c.head, generator=g) * 80).clamp(-448, 448).to(FP8)
            flat[:kv] = x.view(torch.uint8)
            s = torch.randint(*c.steps, (count * per_page, c.kv_heads), generator=g).float().exp2()
            if c.odd_scales:
                s *= 1 + torch.rand(s.shape, generator=g)
            first = max(0, kv - n - c.window + 1) if c.window else 0
            flat[:first] = NAN_CODE  # rows below every token's window were given up
            keys[b].append((x.double(), s.repeat_interleave(c.block, 0)[:kv].double()))
            s[:first // c.block] = math.inf
            s[-(-kv // c.block):] = math.nan
            codes[ids] = flat.view(count, c.page, c.kv_heads, c.head)
            scales[ids] = s.view(count, per_page, c.kv_heads)
        codes, scales = codes.to(device), scales.to(device)
        if c.layout == "hnd":
            codes = codes.transpose(1, 2).contiguous().transpose(1, 2)
            scales = scales.transpose(1, 2).contiguous().transpose(1, 2)
        tensors[name + "_cache"], tensors[name + "_scale"] = codes.view(FP8), scales
    if c.q_slice:
        wide = torch.full((total, c.q_heads + 2, c.head), math.nan, dtype=c.dtype)
        wide[:, 1:-1] = q
        qd = wide.to(device)[:, 1:-1]
    else:
        qd = q.to(device)
    starts = [0]
    for n, _ in c.pairs:
        starts.append(starts[-1] + n)
    c.t = dict(q=qd, block_table=table.to(device),
               kv_len=torch.tensor([kv for _, kv in c.pairs], dtype=torch.int32, device=device),
               cu_q=torch.tensor(starts, dtype=torch.int32, device=device) if c.cu else None,
               max_q=max([n for n, _ in c.pairs] + [1]), **tensors)
    return q, keys


def reference(c: Fp8Case, q, keys):
    """(out, bound, lse) in 64 bits."""
    G = c.q_heads // c.kv_heads
    scale = c.head ** -0.5 if c.scale is None else c.scale
    out = torch.zeros(q.shape, dtype=torch.float64)
    bound = torch.zeros(q.shape, dtype=torch.float64)
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64)
    at = 0
    for (n, kv), ((kc, ks), (vc, vs)) in zip(c.pairs, keys):
        rows = slice(at, at + n)
        at += n
        if n == 0 or kv == 0:
            continue
        place, j = torch.arange(kv - n, kv)[:, None], torch.arange(kv)
        seen = torch.ones(n, kv, dtype=torch.bool)
        if c.causal:
            seen &= j <= place
        if c.window:
            seen &= j > place - c.window
        for h in range(c.q_heads):
            g = h // G
            s = q[rows, h].double() @ (kc[:, g] * ks[:, g, None]).t() * scale
            s = s.masked_fill(~seen, -math.inf)
            top = s.amax(-1, keepdim=True).clamp_min(-1e300)
            p = (s - top).exp()
            l = p.sum(-1, keepdim=True)
            live = l > 0
            w = torch.where(live, p / torch.where(live, l, 1.0), 0.0)
            v = vc[:, g] * vs[:, g, None]
            o, a = w @ v, w @ v.abs()
            e = U[c.dtype] * o.abs() + (2.0 ** -11 + 2.0 ** -13) * a
            e += 2.0 ** -25 * (w * vs[:, g]).amax(1, keepdim=True) * (seen.double() @ vc[:, g].abs())
            if c.dtype == torch.float16:
                e += 2.0 ** -25
            out[rows, h], bound[rows, h] = o, e
            lse[rows, h] = torch.where(live, top + l.log(), -math.inf).squeeze(-1)
    return out, bound * 1.01 + 1e-30, lse


def scale_for(top: torch.Tensor) -> torch.Tensor:
    """The smallest power of two, within its limits, that 448 times is no smaller than ``top``."""
    s = torch.full_like(top, 2.0 ** -40)
    for e in range(-40, 40):
        s = torch.where(top > 448 * 2.0 ** e, torch.full_like(top, 2.0 ** (e + 1)), s)
    return s


def append(x, cache, scale, slots):
    """One cache and its scales after a call that writes x [tokens, heads, D] (float32), on the CPU, block
    by block; of two tokens with one slot the later."""
    pages, page, heads, D = cache.shape
    block = page // scale.shape[1]
    cache, scale = cache.clone(), scale.clone()
    flat, flat_scale = cache.view(torch.uint8).view(-1, block, heads, D), scale.view(-1, heads)
    at = {}
    for t, s in enumerate(slots.tolist()):
        if 0 <= s < pages * page:
            at.setdefault(s // block, {})[s % block] = t
    for b, rows in at.items():
        new = x[list(rows.values())]
        top = new.abs().nan_to_num(nan=0.0, posinf=math.inf).amax((0, 2))
        fit, old = scale_for(top), flat_scale[b].clone()
        so_far = torch.zeros_like(old)
        if 0 not in rows:
            good = (old > 0) & torch.isfinite(old)
            up = torch.where(good, old, 1.0).clamp(2.0 ** -40, 2.0 ** 40)
            so_far = torch.where(good, torch.exp2(torch.ceil(torch.log2(up.double()))).float(), 0.0)
        now = torch.maximum(fit, so_far)
        f = torch.where((so_far > 0) & (now != old), old / now, 1.0)
        for r in range(max(rows)):
            if r in rows or 0 in rows:
                continue
            row = flat[b, r].view(FP8).float() * f[:, None]
            moved = (f != 1)[:, None].expand_as(row)
            flat[b, r] = torch.where(moved, to_e4m3(row), flat[b, r])
        for r, t in rows.items():
            flat[b, r] = to_e4m3(x[t] / now[:, None])
        flat_scale[b] = now
    return cache, scale


def to_e4m3(x):
    """Bytes of e4m3, past its largest number that one."""
    return torch.where(x.isnan(), x, x.clamp(-448, 448)).to(FP8).view(torch.uint8)


def turned(x, positions, table, pairs, sections=None, order="blocks"):
    """x [tokens, heads, D] turned by its positions, in 32 bits."""
    half = table.shape[1] // 2
    positions = (positions if positions.dim() == 2 else positions[None]).long()
    axis = []
    for i in range(half):
        if positions.shape[0] == 1:
            axis.append(0)
        elif order == "blocks":
            ends = torch.tensor(sections).cumsum(0)
            axis.append(int((i >= ends).sum()))
        else:
            a = i % positions.shape[0]
            axis.append(a if i // positions.shape[0] < sections[a] else 0)
    row = positions[axis].t()  # [tokens, half]
    bad = (row < 0) | (row >= table.shape[0])
    row = row.clamp(0, table.shape[0] - 1)
    col = torch.arange(half)
    cos = torch.where(bad, math.nan, table[row, col])[:, None]
    sin = torch.where(bad, math.nan, table[row, col + half])[:, None]
    x = x.float().clone()
    if pairs == "half":
        a, b = x[..., :half].clone(), x[..., half:2 * half].clone()
        x[..., :half], x[..., half:2 * half] = a * cos - b * sin, b * cos + a * sin
    else:
        a, b = x[..., 0:2 * half:2].clone(), x[..., 1:2 * half:2].clone()
        x[..., 0:2 * half:2], x[..., 1:2 * half:2] = a * cos - b * sin, b * cos + a * sin
    return x
