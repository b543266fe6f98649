"""The operators of an 8-bit paged cache, as measured cases.

A decoder layer that keeps its keys and values in 8 bits (e4m3, with one float32 scale for each block
of tokens and kv head) holds twice the context in the same memory and reads half the bytes per step.
The cases are the three operators that work on such a cache:

* ``append``     rotary positions for q and k, k and v rounded into their blocks of the cache; a
                 block whose scale grows has its older tokens rounded again
* ``attention``  softmax(scale q k^T) v of the new tokens over their sequences' 8-bit pages, causal
* ``pages``      copies of whole pages of every layer's caches and scales, as forking a sequence and
                 compacting the cache need them

``own`` picks between the plain form (elementary tensor operations in 32 bits) and the package's
entry points. Head counts, head sizes and page sizes are the usual ones of a serving cache.

The scale of a block and head that a call writes to, with A the largest absolute value that it
writes there and 2^e the smallest power of two with A <= 448 * 2^e (-40 <= e <= 40): 2^e where the
call writes the block's first token, else the larger of 2^e and the scale so far.
"""
import math
import os
import random
import sys

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "e4m3": torch.float8_e4m3fn}
_BYTES = {"bf16": 2, "f16": 2, "e4m3": 1}
_TOP = 448.0  # the largest e4m3 value


def _package():
    """The package, imported at the first call that needs it (module attribute afterwards)."""
    global _ftb
    try:
        return _ftb
    except NameError:
        sys.path.insert(0, os.path.abspath("freetoken-ox-boost_b200"))
        import ftb as _ftb
        return _ftb


# ---- cases -----------------------------------------------------------------------------------


def listed():
    return [
        # one decode step of a batch: each token joins the last block of its own sequence
        dict(name="append_decode", op="append", batch=64, new=1, past=4000, q_heads=32, kv_heads=8,
             head=128, rot=128, pairs="half", page=64, block=64, type="bf16", mix=11),
        # chunks of a few ragged sequences, a partial rotation, small blocks, f16
        dict(name="append_ragged", op="append", batch=7, new=230, past=500, q_heads=12, kv_heads=4,
             head=80, rot=48, pairs="adjacent", page=32, block=16, type="f16", mix=12),
        # a prefill step: three long prompts
        dict(name="append_prefill", op="append", batch=3, new=8190, past=0, q_heads=32, kv_heads=8,
             head=128, rot=128, pairs="half", page=64, block=64, type="bf16", mix=13),
        # one request, one new token, a short chat: pure latency
        dict(name="attn8_one_token", op="attention", batch=1, new=1, kv=901, ragged=False, pad=0,
             q_heads=32, kv_heads=8, head=128, page=16, block=16, window=0, lse=False, type="bf16",
             mix=21),
        # a decode batch of a server: ragged contexts up to 8K, some slots of the batch unused
        dict(name="attn8_decode", op="attention", batch=64, new=1, kv=8192, ragged=True, pad=3,
             q_heads=32, kv_heads=8, head=128, page=64, block=64, window=0, lse=False, type="bf16",
             mix=22),
        # few requests with long documents: the cache is far larger than the on-chip memory
        dict(name="attn8_decode_long", op="attention", batch=3, new=1, kv=131072, ragged=True,
             pad=0, q_heads=32, kv_heads=8, head=128, page=128, block=128, window=0, lse=False,
             type="bf16", mix=23),
        # continuous batching: chunks of different lengths, decode tokens among them, a sliding
        # window, groups of three heads, and the log sum for merging with another part
        dict(name="attn8_mixed_window", op="attention", batch=12, new=300, kv=2900, ragged=True,
             pad=1, q_heads=24, kv_heads=8, head=64, page=32, block=32, window=1000, lse=True,
             type="f16", mix=24),
        # whole prompts packed without a context before them
        dict(name="attn8_prompts", op="attention", batch=8, new=2048, kv=0, ragged=True, pad=0,
             q_heads=32, kv_heads=8, head=128, page=64, block=64, window=0, lse=False, type="bf16",
             mix=25),
        # a prefill chunk late in a long document
        dict(name="attn8_long_chunk", op="attention", batch=1, new=4093, kv=32771, ragged=False,
             pad=0, q_heads=32, kv_heads=8, head=128, page=64, block=64, window=0, lse=False,
             type="bf16", mix=26),
        # sequences forked for sampling: the last, half-filled page of each gets a copy
        dict(name="pages_fork", op="pages", layers=4, count=5, kv_heads=8, head=128, page=64,
             block=64, type="e4m3"),
        # a small 16-bit cache of odd heads tidied up
        dict(name="pages_compact_small", op="pages", layers=2, count=301, kv_heads=3, head=80,
             page=16, block=0, type="bf16"),
        # a server's cache compacted between two bursts
        dict(name="pages_compact", op="pages", layers=8, count=1000, kv_heads=8, head=128, page=64,
             block=64, type="e4m3"),
    ]


def _log_int(rng, low, high):
    """An integer spread over the logarithm of [low, high]."""
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _draw_block(rng):
    page = rng.choice([16, 32, 64, 128])
    return dict(page=page, block=rng.choice([b for b in (16, 32, 64, 128) if b <= page]))


def _draw_append(rng):
    head = rng.choice([64, 80, 112, 128, 128])
    kv_heads = rng.choice([1, 2, 4, 8])
    tokens = _log_int(rng, 1, 16384)
    batch = rng.choice([tokens, _log_int(rng, 1, min(tokens, 64))])  # a decode step, or chunks
    return dict(op="append", batch=batch, new=-(-tokens // batch),
                past=rng.choice([0, _log_int(rng, 1, max(1, min(16384, 262144 // batch)))]),
                q_heads=kv_heads * rng.choice([2, 5, 7, 8]), kv_heads=kv_heads, head=head,
                rot=rng.choice([head, head, head // 2 // 8 * 8]),
                pairs=rng.choice(["half", "adjacent"]), type=rng.choice(["bf16", "f16"]),
                mix=rng.randrange(1 << 30), **_draw_block(rng))


def _draw_attention(rng):
    head = rng.choice([64, 80, 112, 128, 128])
    kv_heads = rng.choice([1, 2, 4, 8])
    shape = dict(q_heads=kv_heads * rng.choice([1, 2, 4, 5, 7, 8]), kv_heads=kv_heads, head=head,
                 type=rng.choice(["bf16", "f16"]), ragged=rng.random() < 0.7,
                 window=rng.choice([0, 0, _log_int(rng, 64, 8192)]), lse=rng.random() < 0.3,
                 mix=rng.randrange(1 << 30), **_draw_block(rng))
    kind = rng.choice(["decode", "chunk", "prompt"])
    if kind == "decode":
        batch = _log_int(rng, 1, 128)
        return dict(op="attention", batch=batch, new=1, pad=rng.choice([0, 0, 1]),
                    kv=_log_int(rng, 16, min(131072, 524288 // batch)), **shape)
    batch = _log_int(rng, 1, 16)
    new = _log_int(rng, 2, 4096 // batch)
    kv = 0 if kind == "prompt" else _log_int(rng, new, min(32768, 65536 // batch))
    return dict(op="attention", batch=batch, new=new, kv=kv, pad=rng.choice([0, 0, 1]), **shape)


def _draw_pages(rng):
    return dict(op="pages", layers=_log_int(rng, 1, 12), count=_log_int(rng, 1, 2000),
                kv_heads=rng.choice([1, 2, 3, 8]), head=rng.choice([64, 80, 112, 128]),
                **rng.choice([dict(_draw_block(rng), type="e4m3"),
                              dict(page=rng.choice([8, 16, 64]), block=0, type="f16")]))


def draw(rng):
    largest = max(_seconds(work(c)) for c in listed())
    moved = max(work(c)["bytes"] for c in listed() if c["op"] == "pages")
    while True:
        case = rng.choice([_draw_append, _draw_attention, _draw_attention, _draw_pages])(rng)
        # no more work than the largest listed case, no more scores than its plain form holds, no
        # more pages moved than by the largest of those
        if _seconds(work(case)) <= largest and _scores(case) <= 32 * 4093 * 32771 and (
                case["op"] != "pages" or work(case)["bytes"] <= moved):
            return case


def _seconds(w):
    return max(w["bytes"] / 6e12, w["flops"] / 1.5e15)


def _scores(case):
    if case["op"] != "attention":
        return 0
    pairs = _lengths(case)
    return case["q_heads"] * len(pairs) * max(n for n, _ in pairs) * max(n for _, n in pairs)


def _lengths(case):
    """(new tokens, length of the sequence with them) of each sequence of an attention case. They go
    by the case alone; padded entries of the batch have one new token and no keys."""
    rng = random.Random(case["mix"])
    new, kv, out = case["new"], case["kv"], []
    for b in range(case["batch"]):
        n = new if not case["ragged"] or new == 1 or b == 0 else _log_int(rng, 1, new)
        # kv == 0: a prompt with nothing before it
        total = n if kv == 0 else kv if not case["ragged"] or b == 0 else _log_int(
            rng, max(1, kv // 16), kv)
        out.append((n, max(n, total)))
    pad = min(case["pad"], case["batch"] - 1)
    return out[:len(out) - pad] + [(1, 0)] * pad


def _chunks(case):
    """(tokens before, new tokens) of each sequence of an append case."""
    rng = random.Random(case["mix"])
    new, past = case["new"], case["past"]
    return [(rng.randint(0, past), new if b == 0 else rng.randint((new + 1) // 2, new))
            for b in range(case["batch"])]


def work(case):
    size = _BYTES[case["type"]]
    kv_heads, head = case["kv_heads"], case["head"]
    if case["op"] == "append":
        tokens = sum(n for _, n in _chunks(case))
        # q in and out, k and v in and as bytes into the cache, cos and sin, slot and position; the
        # scales of the blocks written to
        per = (2 * case["q_heads"] + 2 * kv_heads) * head * size + 2 * kv_heads * head + (
            4 * case["rot"] + 8 + 4)
        blocks = sum((p + n - 1) // case["block"] - p // case["block"] + 1 for p, n in _chunks(case))
        return {"bytes": tokens * per + blocks * 2 * kv_heads * 4,
                "flops": tokens * (3.0 * (case["q_heads"] + kv_heads) * case["rot"]
                                   + 4.0 * kv_heads * head)}
    if case["op"] == "pages":
        row = 2 * kv_heads * head * size * case["page"]
        if case["block"]:
            row += 2 * kv_heads * 4 * (case["page"] // case["block"])
        return {"bytes": 2 * case["layers"] * case["count"] * row + 8 * case["count"], "flops": 0}
    heads, window = case["q_heads"], case["window"]
    total = seen = keys = 0
    for n, kv in _lengths(case):
        total += n
        if kv:
            first = kv - n + 1  # keys that the first new token sees, before the window
            cut = lambda m: min(m, window) if window else m  # noqa: E731
            seen += sum(cut(first + i) for i in range(n))
            keys += kv - max(0, first - window) if window else kv
    return {"bytes": 2 * total * heads * head * size + 2 * keys * kv_heads * head
            + 2 * -(-keys // case["block"]) * kv_heads * 4 + (4 * total * heads if case["lse"] else 0),
            "flops": 4.0 * heads * head * seen}


# ---- inputs ----------------------------------------------------------------------------------


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    kind = _TYPES[case["type"]]

    def normal(*shape, dtype=kind, scale=1.0):
        t = torch.empty(*shape, dtype=dtype, device="cuda").normal_(0, 1, generator=gen)
        return t if scale == 1.0 else t.mul_(scale)

    def codes(*shape):
        """e4m3 numbers as a block holds them: most of its range in use."""
        return normal(*shape, dtype=torch.bfloat16, scale=80.0).clamp_(-_TOP, _TOP).to(
            torch.float8_e4m3fn)

    def scales(pages):
        """Powers of two as normal keys and values have them, some a step lower."""
        at = torch.randint(-8, -5, (pages, case["page"] // case["block"], case["kv_heads"]),
                           generator=gen, device="cuda")
        return torch.exp2(at.float())

    state = {"op": case["op"], "case": dict(case)}
    if case["op"] == "pages":
        count, pages = case["count"], 2 * case["count"] + 3
        shape = (pages, case["page"], case["kv_heads"], case["head"])
        state["caches"] = []
        for _ in range(2 * case["layers"]):
            state["caches"].append(codes(*shape) if case["type"] == "e4m3" else normal(*shape))
            if case["block"]:
                state["caches"].append(scales(pages))
        order = torch.randperm(pages, generator=gen, device="cuda", dtype=torch.int32)
        state["src"], state["dst"] = order[:count].contiguous(), order[-count:].contiguous()
        return state
    heads, kv_heads, head, page = case["q_heads"], case["kv_heads"], case["head"], case["page"]
    if case["op"] == "append":
        pairs = _chunks(case)
        rows = sum(n for _, n in pairs)
        need = [-(-(p + n) // page) for p, n in pairs]
        # the projection's output: q, k and v of a token are slices of one row
        qkv = normal(rows, (heads + 2 * kv_heads) * head)
        q, k, v = qkv.split([heads * head, kv_heads * head, kv_heads * head], dim=1)
        state["q"] = q.unflatten(1, (heads, head))
        state["k"] = k.unflatten(1, (kv_heads, head))
        state["v"] = v.unflatten(1, (kv_heads, head))
        # of each sequence only the pages that the new tokens reach are in this cache
        first = [p // page for p, _ in pairs]
        used = sum(n - f for n, f in zip(need, first))
        order = torch.randperm(used + 1, generator=gen, device="cuda")
        lengths = torch.tensor(pairs, device="cuda")
        begin = torch.tensor([0] + [n - f for n, f in zip(need, first)], device="cuda").cumsum(0)
        seq = torch.repeat_interleave(torch.arange(len(pairs), device="cuda"), lengths[:, 1])
        at = torch.arange(rows, device="cuda") - (lengths[:, 1].cumsum(0) - lengths[:, 1])[seq]
        place = lengths[seq, 0] + at
        inner = place // page - lengths[seq, 0] // page
        state["slots"] = order[begin[seq] + inner] * page + place % page
        state["positions"] = place.int()
        span = max(p + n for p, n in pairs)
        state["k_cache"], state["v_cache"] = (codes(used + 1, page, kv_heads, head) for _ in "kv")
        state["k_scale"], state["v_scale"] = scales(used + 1), scales(used + 1)
        half = case["rot"] // 2
        angle = torch.arange(span, device="cuda", dtype=torch.float64)[:, None] * 10000.0 ** (
            -torch.arange(half, device="cuda", dtype=torch.float64) / half)
        state["table"] = torch.cat([angle.cos(), angle.sin()], 1).float()
        return state
    pairs = _lengths(case)
    total = sum(n for n, _ in pairs)
    width = max(1, max(-(-kv // page) for _, kv in pairs))
    used = sum(-(-kv // page) for _, kv in pairs)
    state["k_cache"], state["v_cache"] = (codes(used + 1, page, kv_heads, head) for _ in "kv")
    state["k_scale"], state["v_scale"] = scales(used + 1), scales(used + 1)
    order = torch.randperm(used + 1, generator=gen, device="cuda", dtype=torch.int32)
    table = torch.zeros(len(pairs), width, dtype=torch.int32, device="cuda")
    at = 0
    for b, (_, kv) in enumerate(pairs):  # pages in an order that has nothing to do with the sequence
        count = -(-kv // page)
        table[b, :count] = order[at:at + count]
        at += count
    state["block_table"] = table
    state["q"] = normal(total, heads, head)
    state["kv_len"] = torch.tensor([kv for _, kv in pairs], dtype=torch.int32, device="cuda")
    starts = [0]
    for n, _ in pairs:
        starts.append(starts[-1] + n)
    state["max_new"] = max(n for n, _ in pairs)
    # a decode step has one token in each sequence, and no list of their starts
    state["starts"] = None if state["max_new"] == 1 else torch.tensor(starts, dtype=torch.int32,
                                                                      device="cuda")
    return state


# ---- one pass --------------------------------------------------------------------------------


def run(state):
    return _run_own(state) if own else _PLAIN[state["op"]](state)


def _run_own(s):
    ftb, case = _package(), s["case"]
    if s["op"] == "append":
        q = ftb.rope_append(s["q"], s["k"], s["v"], s["positions"], s["table"], s["k_cache"],
                            s["v_cache"], s["slots"], pairs=case["pairs"], k_scale=s["k_scale"],
                            v_scale=s["v_scale"])
        return {"q": q, **{n: s[n] for n in ("k_cache", "v_cache", "k_scale", "v_scale")}}
    if s["op"] == "pages":
        ftb.copy_pages(s["caches"], s["src"], s["dst"])
        return s["caches"]
    r = ftb.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["block_table"], s["kv_len"],
                            s["starts"], s["max_new"], window=case["window"],
                            return_lse=case["lse"], k_scale=s["k_scale"], v_scale=s["v_scale"])
    return {"out": r[0], "lse": r[1]} if case["lse"] else {"out": r}


def _rotate(x, cos, sin, case):
    rot, half = case["rot"], case["rot"] // 2
    x = x.float()
    part, rest = x[..., :rot], x[..., rot:]
    if case["pairs"] == "half":
        a, b = part[..., :half], part[..., half:]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    else:
        a, b = part[..., 0::2], part[..., 1::2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    return torch.cat([turned, rest], -1)


def _plain_append(s):
    case, half = s["case"], s["case"]["rot"] // 2
    row = s["table"][s["positions"].long()]
    cos, sin = row[:, None, :half], row[:, None, half:]
    size, per_page = case["block"], case["page"] // case["block"]
    blocks, index = torch.unique(s["slots"] // size, return_inverse=True)
    at = s["slots"] % size
    new = torch.zeros(len(blocks), size, dtype=torch.bool, device=at.device)
    new[index, at] = True
    rows = torch.arange(size, device=at.device)
    older = ~new & (rows < (new * rows).amax(1, keepdim=True)) & ~new[:, :1]
    page, part = blocks // per_page, blocks % per_page
    for name, x in (("k", _rotate(s["k"], cos, sin, case)), ("v", s["v"].float())):
        cache, scale = s[name + "_cache"], s[name + "_scale"]
        whole = cache.view(cache.shape[0], per_page, size, *cache.shape[2:])
        old = scale[page, part]  # [blocks, heads]
        top = torch.zeros_like(old).index_reduce_(0, index, x.abs().amax(-1), "amax")
        mantissa, power = torch.frexp(top / _TOP)
        power = torch.where(top == 0, -40, torch.where(mantissa == 0.5, power - 1, power))
        fit = torch.exp2(power.clamp(-40, 40).float())
        now = torch.where(new[:, :1], fit, torch.maximum(old, fit))
        held = whole[page, part].float() * (old / now)[:, None, :, None]
        held[index, at] = x / now[index][..., None]
        held = torch.where((new | older)[..., None, None], held, whole[page, part].float())
        whole[page, part] = held.to(cache.dtype)
        scale[page, part] = now
    return {"q": _rotate(s["q"], cos, sin, case).to(s["q"].dtype),
            **{n: s[n] for n in ("k_cache", "v_cache", "k_scale", "v_scale")}}


def _plain_pages(s):
    src, dst = s["src"].long(), s["dst"].long()
    for cache in s["caches"]:
        held = cache.view(torch.uint8) if cache.dtype == torch.float8_e4m3fn else cache
        held[dst] = held[src]
    return s["caches"]


def _gathered(s, name):
    """[batch, kv heads, keys, head] of every sequence's pages, as the numbers they stand for."""
    case, table = s["case"], s["block_table"].long()
    x = s[name + "_cache"][table].float()  # [batch, width, page, heads, head]
    x = x.unflatten(2, (-1, case["block"])) * s[name + "_scale"][table][:, :, :, None, :, None]
    return x.flatten(1, 3).transpose(1, 2)


def _plain_attention(s):
    case, q, kv_len = s["case"], s["q"], s["kv_len"].long()
    batch, new, heads, head = kv_len.numel(), s["max_new"], case["q_heads"], case["head"]
    kv_heads, group = case["kv_heads"], case["q_heads"] // case["kv_heads"]
    token = torch.arange(q.shape[0], device=q.device)
    starts = (torch.arange(batch + 1, device=q.device) if s["starts"] is None
              else s["starts"].long())
    row = torch.searchsorted(starts, token, right=True) - 1  # the sequence of each token
    at = token - starts[row]
    padded = torch.zeros(batch, new, heads, head, dtype=torch.float32, device=q.device)
    padded[row, at] = q.float()
    # [batch, kv head, group * new, head] against [batch, kv head, keys, head]
    padded = padded.view(batch, new, kv_heads, group, head).permute(0, 2, 3, 1, 4)
    padded = padded.reshape(batch, kv_heads, group * new, head)
    score = torch.matmul(padded, _gathered(s, "k").transpose(2, 3)).mul_(head ** -0.5)
    score = score.view(batch, kv_heads, group, new, -1)
    key = torch.arange(score.shape[-1], device=q.device)
    # the position of each new token in its sequence
    place = (kv_len - starts.diff())[:, None] + torch.arange(new, device=q.device)
    hidden = (key > place[..., None]) | (key >= kv_len[:, None, None])
    if case["window"]:
        hidden |= key <= place[..., None] - case["window"]
    score.masked_fill_(hidden[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True).clamp_min(-3e38)
    score = score.sub_(top).exp_()
    total = score.sum(-1, keepdim=True)
    out = torch.matmul(score.view(batch, kv_heads, group * new, -1), _gathered(s, "v"))
    out = out.view(batch, kv_heads, group, new, head) / torch.where(total > 0, total, 1.0)
    out = out.permute(0, 3, 1, 2, 4).reshape(batch, new, heads, head)[row, at].to(q.dtype)
    if not case["lse"]:
        return {"out": out}
    lse = (top + total.log()).squeeze(-1)
    return {"out": out, "lse": lse.permute(0, 3, 1, 2).reshape(batch, new, heads)[row, at]}


_PLAIN = {"append": _plain_append, "pages": _plain_pages, "attention": _plain_attention}


# ---- the definition in 64 bits ---------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "pages": _exact_pages, "attention": _exact_attention}[
        case["op"]](s)


def _exact_append(s):
    case = s["case"]
    half, size, page = case["rot"] // 2, case["block"], case["page"]
    angle = s["table"].double()[s["positions"].long()]
    turn = torch.complex(angle[:, :half], angle[:, half:])  # cos + i sin
    first = torch.arange(half, device="cuda") * (1 if case["pairs"] == "half" else 2)
    second = first + (half if case["pairs"] == "half" else 1)

    def rotate(x):
        x = x.double().clone()
        z = torch.complex(x[..., first], x[..., second]) * turn[:, None]
        x[..., first], x[..., second] = z.real, z.imag
        return x

    out = {"q": rotate(s["q"])}
    n_blocks = s["k_cache"].shape[0] * page // size
    block, row = s["slots"] // size, s["slots"] % size
    last = torch.full((n_blocks,), -1, device="cuda").scatter_reduce(0, block, row, "amax")
    fresh = torch.zeros(n_blocks, dtype=torch.bool, device="cuda")
    fresh[block[row == 0]] = True
    written = torch.zeros(n_blocks, size, dtype=torch.bool, device="cuda")
    written[block, row] = True
    again = torch.arange(size, device="cuda") < last[:, None]
    again &= ~written & ~fresh[:, None]
    for name, x in (("k", rotate(s["k"])), ("v", s["v"].double())):
        old = s[name + "_scale"].double().reshape(n_blocks, -1)
        most = torch.zeros_like(old)
        most.scatter_reduce_(0, block[:, None].expand(-1, old.shape[1]), x.abs().amax(2), "amax")
        fit = torch.exp2(torch.ceil(torch.log2(most / _TOP)).clamp(-40, 40))
        now = torch.where(fresh[:, None], fit, torch.maximum(old, fit))
        now = torch.where(last[:, None] >= 0, now, old)
        held = s[name + "_cache"].double().reshape(n_blocks, size, *x.shape[1:])
        held = torch.where(again[..., None, None], held * (old / now)[:, None, :, None], held)
        held[block, row] = x / now[block][..., None]
        out[name + "_cache"] = held.reshape(s[name + "_cache"].shape)
        out[name + "_scale"] = now.reshape(s[name + "_scale"].shape)
    return out


def _exact_pages(s):
    out = []
    for cache in s["caches"]:
        held = cache.double()
        out.append(held.index_copy(0, s["dst"].long(), held.index_select(0, s["src"].long())))
    return out


def _exact_attention(s):
    case = s["case"]
    page, size, window = case["page"], case["block"], case["window"]
    group = case["q_heads"] // case["kv_heads"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.full(s["q"].shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    begin = 0
    for b, (n, kv) in enumerate(_lengths(case)):
        rows = slice(begin, begin + n)
        begin += n
        if kv == 0:
            continue
        at = torch.arange(kv, device="cuda")
        ids = s["block_table"][b].long()[at // page]
        place = torch.arange(kv - n, kv, device="cuda")[:, None]
        seen = at <= place
        if window:
            seen &= at > place - window
        for g in range(case["kv_heads"]):
            k, v = (s[x + "_cache"][ids, at % page, g].double()
                    * s[x + "_scale"][ids, at % page // size, g, None].double() for x in "kv")
            for h in range(g * group, (g + 1) * group):
                score = s["q"][rows, h].double() @ k.t() / math.sqrt(case["head"])
                score[~seen] = -math.inf
                lse[rows, h] = torch.logsumexp(score, 1)
                out[rows, h] = torch.softmax(score, 1) @ v
    return {"out": out, "lse": lse} if case["lse"] else {"out": out}
