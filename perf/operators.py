"""The operators around the MoE layer of a decoder block, as measured cases.

A decoder block that uses this package's experts runs, per layer: the norm before its attention,
the rotary embedding of the new tokens' queries and keys with the write into the paged cache, the
attention of those tokens over the cache, the norms after the attention and before the MoE layer
with the gated residual. The cases here are those three operators:

* ``norm``       r = x + scale * gate * rms(y) * post;  h = rms(r) * pre
* ``rope``       rotary positions on one or three axes for q and k, k and v into their cache slots
* ``attention``  softmax(scale q k^T) v of the new tokens over their sequence's pages, causal

``own`` picks between the plain form (elementary tensor operations in 32 bits) and the package's
entry points. Sizes: hidden 4096 and 2048 are the package's own layer shapes, head counts, head
sizes and page sizes are the usual ones of a serving cache.
"""
import math
import os
import random
import sys

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_BYTES = {"bf16": 2, "f16": 2, "f32": 4}


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
        # one token of one request between two blocks of a layer: pure latency
        dict(name="norm_one_token", op="norm", tokens=1, hidden=4096, type="bf16",
             residual="bf16", gate="none", post=True),
        # a prefill chunk with the residual stream kept in 32 bits and a gate per token
        dict(name="norm_prefill", op="norm", tokens=4096, hidden=4096, type="bf16",
             residual="f32", gate="token", post=True),
        # a ragged batch at a width that fills no vector, f16, with a full gate
        dict(name="norm_odd_width", op="norm", tokens=1021, hidden=2045, type="f16",
             residual="f16", gate="full", post=True),
        # a decode batch of text: one new token per sequence, one position axis
        dict(name="rope_decode", op="rope", tokens=64, q_heads=32, kv_heads=8, head=128,
             rot=128, axes=1, order="blocks", pairs="half", page=64, type="bf16"),
        # a partial rotation of adjacent pairs, odd token count, head size not a power of two
        dict(name="rope_partial", op="rope", tokens=777, q_heads=12, kv_heads=4, head=80,
             rot=48, axes=1, order="blocks", pairs="adjacent", page=32, type="f16"),
        # the tokens of images in a prefill chunk: time, height and width, frequencies dealt in turn
        dict(name="rope_images", op="rope", tokens=8190, q_heads=32, kv_heads=8, head=128,
             rot=128, axes=3, order="cyclic", pairs="half", page=16, type="bf16"),
        # one request, one new token, a short chat: pure latency
        dict(name="attn_one_token", op="attention", batch=1, new=1, kv=777, ragged=False, pad=0,
             q_heads=32, kv_heads=8, head=128, page=16, window=0, lse=False, type="bf16", mix=1),
        # a decode batch of a server: ragged contexts up to 8K, some slots of the batch unused
        dict(name="attn_decode", op="attention", batch=64, new=1, kv=8192, ragged=True, pad=3,
             q_heads=32, kv_heads=8, head=128, page=64, window=0, lse=False, type="bf16", mix=2),
        # few requests with long documents: the cache is far larger than the on-chip memory
        dict(name="attn_decode_long", op="attention", batch=3, new=1, kv=131072, ragged=True,
             pad=0, q_heads=32, kv_heads=8, head=128, page=64, window=0, lse=False, type="bf16",
             mix=3),
        # continuous batching: chunks of different lengths, decode tokens among them, a sliding
        # window, groups of three heads, and the log sum for merging with another part
        dict(name="attn_mixed_window", op="attention", batch=12, new=300, kv=3000, ragged=True,
             pad=1, q_heads=24, kv_heads=8, head=64, page=32, window=1000, lse=True, type="f16",
             mix=4),
        # whole prompts packed without a context before them
        dict(name="attn_prompts", op="attention", batch=8, new=2048, kv=0, ragged=True, pad=0,
             q_heads=32, kv_heads=8, head=128, page=64, window=0, lse=False, type="bf16", mix=5),
        # a prefill chunk late in a long document
        dict(name="attn_long_chunk", op="attention", batch=1, new=4093, kv=32771, ragged=False,
             pad=0, q_heads=32, kv_heads=8, head=128, page=64, window=0, lse=False, type="bf16",
             mix=6),
    ]


def _log_int(rng, low, high):
    """An integer spread over the logarithm of [low, high]."""
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _draw_norm(rng):
    tokens = _log_int(rng, 1, 8192)
    hidden = rng.choice([_log_int(rng, 64, 8192) | 1, 16 * _log_int(rng, 4, 511) + 8, 2048, 4096])
    kind = rng.choice(["bf16", "bf16", "f16"])
    return dict(op="norm", tokens=tokens, hidden=hidden, type=kind,
                residual=rng.choice([kind, "f32"]),
                gate=rng.choice(["none", "channel", "token", "full"]), post=rng.random() < 0.7)


def _draw_rope(rng):
    head = rng.choice([64, 80, 112, 128, 128])
    kv_heads = rng.choice([1, 2, 4, 8])
    return dict(op="rope", tokens=_log_int(rng, 1, 8192), q_heads=kv_heads * rng.choice([2, 5, 7, 8]),
                kv_heads=kv_heads, head=head, rot=rng.choice([head, head, head // 2 // 8 * 8]),
                axes=rng.choice([1, 3]), order=rng.choice(["blocks", "cyclic"]),
                pairs=rng.choice(["half", "adjacent"]), page=rng.choice([16, 32, 64, 128]),
                type=rng.choice(["bf16", "f16"]))


def _draw_attention(rng):
    head = rng.choice([64, 80, 112, 128, 128])
    kv_heads = rng.choice([1, 2, 4, 8])
    shape = dict(q_heads=kv_heads * rng.choice([1, 2, 4, 5, 7, 8]), kv_heads=kv_heads, head=head,
                 page=rng.choice([16, 32, 64, 128]), type=rng.choice(["bf16", "f16"]),
                 window=rng.choice([0, 0, _log_int(rng, 64, 8192)]), lse=rng.random() < 0.3,
                 ragged=rng.random() < 0.7, mix=rng.randrange(1 << 30))
    kind = rng.choice(["decode", "chunk", "prompt"])
    if kind == "decode":
        batch = _log_int(rng, 1, 128)
        return dict(op="attention", batch=batch, new=1, pad=rng.choice([0, 0, 1]),
                    kv=_log_int(rng, 16, min(131072, 524288 // batch)), **shape)
    batch = _log_int(rng, 1, 16)
    new = _log_int(rng, 2, 4096 // batch)
    kv = 0 if kind == "prompt" else _log_int(rng, new, min(32768, 65536 // batch))
    return dict(op="attention", batch=batch, new=new, kv=kv, pad=rng.choice([0, 0, 1]), **shape)


def draw(rng):
    largest = max(_seconds(work(c)) for c in listed())
    while True:
        case = rng.choice([_draw_norm, _draw_rope, _draw_attention, _draw_attention])(rng)
        # no more work than the largest listed case, no more scores than its plain form holds
        if _seconds(work(case)) <= largest and _scores(case) <= 32 * 4093 * 32771:
            return case


def _seconds(w):
    return max(w["bytes"] / 6e12, w["flops"] / 1.5e15)


def _scores(case):
    if case["op"] != "attention":
        return 0
    pairs = _lengths(case)
    return case["q_heads"] * len(pairs) * max(n for n, _ in pairs) * max(n for _, n in pairs)


def _lengths(case):
    """(new tokens, length of the sequence with them) of each sequence of the batch. They go by the
    case alone; padded entries of the batch have one new token and no keys."""
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


def work(case):
    size = _BYTES[case["type"]]
    if case["op"] == "norm":
        rows, width = case["tokens"], case["hidden"]
        gate = {"none": 0, "channel": width, "token": rows, "full": rows * width}[case["gate"]]
        weights = (2 if case["post"] else 1) * width
        return {"bytes": rows * width * (2 * size + 2 * _BYTES[case["residual"]])
                + (gate + weights) * size,
                "flops": 12.0 * rows * width}
    if case["op"] == "rope":
        row = case["head"] * size
        # q in and out, k and v in and into the cache, cos and sin of the token, slot, positions
        per = 2 * (case["q_heads"] + 2 * case["kv_heads"]) * row + 4 * case["rot"] + 8 + 4 * case["axes"]
        return {"bytes": case["tokens"] * per,
                "flops": 3.0 * case["tokens"] * (case["q_heads"] + case["kv_heads"]) * case["rot"]}
    heads, kv_heads, head, window = case["q_heads"], case["kv_heads"], case["head"], case["window"]
    total = seen = keys = 0
    for n, kv in _lengths(case):
        total += n
        if kv:
            first = kv - n + 1  # keys that the first new token sees, before the window
            cut = lambda m: min(m, window) if window else m  # noqa: E731
            seen += sum(cut(first + i) for i in range(n))
            keys += kv - max(0, first - window) if window else kv
    row = head * size
    return {"bytes": 2 * total * heads * row + 2 * keys * kv_heads * row
            + (4 * total * heads if case["lse"] else 0),
            "flops": 4.0 * heads * head * seen}


# ---- inputs ----------------------------------------------------------------------------------


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    kind = _TYPES[case["type"]]

    def normal(*shape, dtype=kind, scale=1.0, mean=0.0):
        t = torch.empty(*shape, dtype=dtype, device="cuda").normal_(0, 1, generator=gen)
        return t if scale == 1.0 and mean == 0.0 else t.mul_(scale).add_(mean)

    state = {"op": case["op"], "case": dict(case)}
    if case["op"] == "norm":
        rows, width = case["tokens"], case["hidden"]
        state["x"] = normal(rows, width, dtype=_TYPES[case["residual"]], scale=3.0)
        state["y"] = normal(rows, width)
        state["post"] = normal(width, scale=0.1, mean=0.8) if case["post"] else None
        state["pre"] = normal(width, scale=0.1, mean=1.0)
        shape = {"none": None, "channel": (width,), "token": (rows, 1), "full": (rows, width)}
        shape = shape[case["gate"]]
        state["gate"] = normal(*shape, scale=0.3, mean=1.0) if shape else None
        return state
    heads, kv_heads, head, page = case["q_heads"], case["kv_heads"], case["head"], case["page"]
    if case["op"] == "rope":
        rows = case["tokens"]
        # the projection's output: q, k and v of a token are slices of one row
        qkv = normal(rows, (heads + 2 * kv_heads) * head)
        q, k, v = qkv.split([heads * head, kv_heads * head, kv_heads * head], dim=1)
        state["q"] = q.unflatten(1, (heads, head))
        state["k"] = k.unflatten(1, (kv_heads, head))
        state["v"] = v.unflatten(1, (kv_heads, head))
        pages = -(-rows * 5 // 4 // page) + 1
        state["k_cache"] = normal(pages, page, kv_heads, head)
        state["v_cache"] = normal(pages, page, kv_heads, head)
        state["slots"] = torch.randperm(pages * page, generator=gen, device="cuda")[:rows]
        span = 32768
        if case["axes"] == 1:
            state["positions"] = torch.randint(0, span, (rows,), generator=gen, device="cuda",
                                               dtype=torch.int32)
        else:  # image patches: a frame's position in time, rows and columns of its grid
            at = torch.arange(rows, device="cuda", dtype=torch.int32)
            state["positions"] = torch.stack([at // 1024, at // 32 % 32, at % 32]) + int(
                torch.randint(0, 4096, (1,), generator=gen, device="cuda"))
        half = case["rot"] // 2
        angle = torch.arange(span, device="cuda", dtype=torch.float64)[:, None] * 10000.0 ** (
            -torch.arange(half, device="cuda", dtype=torch.float64) / half)
        state["table"] = torch.cat([angle.cos(), angle.sin()], 1).float()
        third = half // 3
        state["sections"] = None if case["axes"] == 1 else (half - 2 * third, third, third)
        return state
    pairs = _lengths(case)
    total = sum(n for n, _ in pairs)
    width = max(1, max(-(-kv // page) for _, kv in pairs))
    used = sum(-(-kv // page) for _, kv in pairs)
    state["k_cache"] = normal(used + 1, page, kv_heads, head)
    state["v_cache"] = normal(used + 1, page, kv_heads, head)
    order = torch.randperm(used + 1, generator=gen, device="cuda", dtype=torch.int32)
    table = torch.zeros(len(pairs), width, dtype=torch.int32, device="cuda")
    at = 0
    for b, (_, kv) in enumerate(pairs):  # pages in an order that has nothing to do with the sequence
        count = -(-kv // page)
        table[b, :count] = order[at:at + count]
        at += count
    state["table"] = table
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
    if s["op"] == "norm":
        r, h = ftb.block_norm(s["x"], s["y"], post_weight=s["post"], gate=s["gate"], scale=0.5,
                              pre_weight=s["pre"], eps=1e-6)
        return {"residual": r, "normed": h}
    if s["op"] == "rope":
        q = ftb.rope_append(s["q"], s["k"], s["v"], s["positions"], s["table"], s["k_cache"],
                            s["v_cache"], s["slots"], sections=s["sections"],
                            order=case["order"], pairs=case["pairs"])
        return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    r = ftb.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["kv_len"],
                            s["starts"], s["max_new"], window=case["window"],
                            return_lse=case["lse"])
    return {"out": r[0], "lse": r[1]} if case["lse"] else {"out": r}


def _rms(v, weight):
    v = v * torch.rsqrt(v.square().mean(-1, keepdim=True) + 1e-6)
    return v * weight.float()


def _plain_norm(s):
    y = s["y"].float()
    if s["post"] is not None:
        y = _rms(y, s["post"])
    if s["gate"] is not None:
        y = y * s["gate"].float()
    r = s["x"].float() + 0.5 * y
    return {"residual": r.to(s["x"].dtype), "normed": _rms(r, s["pre"]).to(s["y"].dtype)}


def _axis_of(case, sections, device):
    """The position axis of each frequency: a block of frequencies for each axis, or the axes in
    turn (time, height, width, time, ...) for as long as an axis has frequencies left, and time for
    the rest."""
    half = case["rot"] // 2
    i = torch.arange(half, device=device)
    if sections is None:
        return torch.zeros_like(i)
    if case["order"] == "blocks":
        return (i >= sections[0]).long() + (i >= sections[0] + sections[1]).long()
    turn = i % 3
    left = torch.where(turn == 1, 3 * sections[1], 3 * sections[2])
    return torch.where(i < left, turn, 0)


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


def _plain_rope(s):
    case, half = s["case"], s["case"]["rot"] // 2
    positions = s["positions"].long().reshape(case["axes"], -1)
    axis = _axis_of(case, s["sections"], positions.device)
    at = positions[axis].t()  # [tokens, half]
    column = torch.arange(half, device=at.device)
    cos, sin = s["table"][at, column][:, None], s["table"][at, column + half][:, None]
    page = s["slots"] // case["page"], s["slots"] % case["page"]
    s["k_cache"][page] = _rotate(s["k"], cos, sin, case).to(s["k"].dtype)
    s["v_cache"][page] = s["v"]
    return {"q": _rotate(s["q"], cos, sin, case).to(s["q"].dtype), "k_cache": s["k_cache"],
            "v_cache": s["v_cache"]}


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
    k = s["k_cache"][s["table"].long()].flatten(1, 2).transpose(1, 2).float()
    score = torch.matmul(padded, k.transpose(2, 3)).mul_(head ** -0.5)
    del k
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
    v = s["v_cache"][s["table"].long()].flatten(1, 2).transpose(1, 2).float()
    out = torch.matmul(score.view(batch, kv_heads, group * new, -1), v)
    out = out.view(batch, kv_heads, group, new, head) / torch.where(total > 0, total, 1.0)
    out = out.permute(0, 3, 1, 2, 4).reshape(batch, new, heads, head)[row, at].to(q.dtype)
    if not case["lse"]:
        return {"out": out}
    lse = (top + total.log()).squeeze(-1)
    return {"out": out, "lse": lse.permute(0, 3, 1, 2).reshape(batch, new, heads)[row, at]}


_PLAIN = {"norm": _plain_norm, "rope": _plain_rope, "attention": _plain_attention}


# ---- the definition in 64 bits ---------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "rope": _exact_rope, "attention": _exact_attention}[case["op"]](s)


def _exact_norm(s):
    x, y = s["x"].double(), s["y"].double()
    norm = lambda v: v / ((v * v).sum(1, keepdim=True) / v.shape[1] + 1e-6).sqrt()  # noqa: E731
    if s["post"] is not None:
        y = norm(y) * s["post"].double()
    gate = 1.0 if s["gate"] is None else s["gate"].double()
    r = x + y * gate / 2
    return {"residual": r, "normed": norm(r) * s["pre"].double()}


def _exact_rope(s):
    case = s["case"]
    rot, half, rows = case["rot"], case["rot"] // 2, case["tokens"]
    positions = s["positions"].reshape(case["axes"], rows)
    left = list(s["sections"] or (half,))
    axis = []
    for i in range(half):
        if case["order"] == "blocks" or len(left) == 1:
            a = next(j for j, n in enumerate(left) if n)
            left[a] -= 1
        else:
            a = i % 3 if i // 3 < s["sections"][i % 3] else 0
        axis.append(a)
    # each pair as a complex number, turned by cos + i sin
    turn = torch.empty(rows, half, dtype=torch.complex128, device="cuda")
    for i, a in enumerate(axis):
        at = positions[a].long()
        turn[:, i] = torch.complex(s["table"][at, i].double(), s["table"][at, half + i].double())
    first = torch.arange(half, device="cuda") * (1 if case["pairs"] == "half" else 2)
    second = first + (half if case["pairs"] == "half" else 1)

    def rotate(x):
        x = x.double().clone()
        z = torch.complex(x[..., first], x[..., second]) * turn[:, None]
        x[..., first], x[..., second] = z.real, z.imag
        return x

    k_cache, v_cache = s["k_cache"].double(), s["v_cache"].double()
    k_cache.view(-1, *k_cache.shape[2:]).index_copy_(0, s["slots"], rotate(s["k"]))
    v_cache.view(-1, *v_cache.shape[2:]).index_copy_(0, s["slots"], s["v"].double())
    return {"q": rotate(s["q"]), "k_cache": k_cache, "v_cache": v_cache}


def _exact_attention(s):
    case = s["case"]
    page, window = case["page"], case["window"]
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
        slot = s["table"][b].long()[at // page] * page + at % page
        place = torch.arange(kv - n, kv, device="cuda")[:, None]
        seen = at <= place
        if window:
            seen &= at > place - window
        for h in range(case["q_heads"]):
            k = s["k_cache"][:, :, h // group].flatten(0, 1)[slot].double()
            v = s["v_cache"][:, :, h // group].flatten(0, 1)[slot].double()
            score = s["q"][rows, h].double() @ k.t() / math.sqrt(case["head"])
            score[~seen] = -math.inf
            lse[rows, h] = torch.logsumexp(score, 1)
            out[rows, h] = torch.softmax(score, 1) @ v
    return {"out": out, "lse": lse} if case["lse"] else {"out": out}
