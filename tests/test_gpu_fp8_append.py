"""ftb.rope_append into an 8-bit cache: q, codes and scales against the rule of tests/fp8_cases.py, codes
and scales bit for bit."""
import math

import pytest
import torch

import ftb
from tests.fp8_cases import FP8, append, turned

pytestmark = pytest.mark.gpu
BF, F16 = torch.bfloat16, torch.float16


def make(tokens, slots, *, heads=(4, 2), D=64, rot=64, page=32, block=16, pages=8, dtype=BF, axes=1,
         pairs="half", seed=0, layout="nhd", spread=1.0, slot_type=torch.int64, scales=(-9, -4),
         sections=None, order="blocks"):
    g = torch.Generator().manual_seed(seed)
    Hq, Hkv = heads
    qkv = (torch.randn(tokens, Hq + 2 * Hkv, D, generator=g) * spread).to(dtype)
    # blocks whose size goes up and down by powers of two
    qkv[:, Hq:] *= torch.randint(-3, 4, (tokens, 2 * Hkv, 1), generator=g).float().exp2().to(dtype)
    positions = torch.randint(0, 500, (axes, tokens) if axes > 1 else (tokens,), generator=g)
    table = ftb.rope_table(500, rot, device="cpu")
    tensors = {}
    for n in "kv":
        codes = torch.randint(0, 256, (pages, page, Hkv, D), generator=g, dtype=torch.uint8)
        codes[codes & 0x7f == 0x7f] = 0  # (no NaN; a test of its own has them)
        scale = torch.randint(*scales, (pages, page // block, Hkv), generator=g).float().exp2()
        tensors[n + "_cache"], tensors[n + "_scale"] = codes, scale
    slots = torch.as_tensor(slots, dtype=slot_type)
    return dict(qkv=qkv, heads=heads, positions=positions, table=table, slots=slots, pairs=pairs,
                sections=sections, order=order, layout=layout, **tensors)


def call(c, device="cuda"):
    """The call's outputs, on the CPU, with the cache tensors that the call was given."""
    t = {}
    for n in ("k_cache", "v_cache", "k_scale", "v_scale"):
        x = c[n].to(device)
        if c["layout"] == "hnd":
            x = x.transpose(1, 2).contiguous().transpose(1, 2)
        t[n] = x.view(FP8) if "cache" in n else x
    q, k, v = c["qkv"].to(device).split([c["heads"][0], c["heads"][1], c["heads"][1]], 1)
    q = ftb.rope_append(q, k, v, c["positions"].to(device), c["table"].to(device), t["k_cache"],
                        t["v_cache"], c["slots"].to(device), sections=c["sections"], order=c["order"],
                        pairs=c["pairs"], k_scale=t["k_scale"], v_scale=t["v_scale"])
    return {"q": q.cpu(), **{n: (x.view(torch.uint8) if "cache" in n else x).cpu() for n, x in t.items()}}


def check(c):
    got = call(c)
    q, k, v = c["qkv"].split([c["heads"][0], c["heads"][1], c["heads"][1]], 1)
    turn = lambda x: turned(x, c["positions"], c["table"], c["pairs"], c["sections"], c["order"])  # noqa: E731
    assert torch.equal(got["q"], turn(q).to(q.dtype)) or torch.equal(
        got["q"].isnan(), turn(q).to(q.dtype).isnan())
    for n, x in (("k", turn(k)), ("v", v.float())):
        codes, scale = append(x, c[n + "_cache"], c[n + "_scale"], c["slots"])
        assert torch.equal(got[n + "_scale"].view(torch.int32), scale.view(torch.int32)), n
        nan = codes & 0x7f == 0x7f
        assert torch.equal(got[n + "_cache"][~nan], codes[~nan]), n
        assert (got[n + "_cache"][nan] & 0x7f == 0x7f).all()
    return got


SIZES = [0, 1, 2, 15, 16, 17, 33, 100]


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("tokens", SIZES)
def test_a_prompt(tokens, dtype):
    check(make(tokens, range(32, 32 + tokens), dtype=dtype, seed=tokens))


@pytest.mark.parametrize("first", [1, 5, 15, 16, 31])
@pytest.mark.parametrize("tokens", [1, 3, 20, 70])
def test_joins_a_block(first, tokens):
    """Blocks that hold older rows, some of whose scales have to grow."""
    check(make(tokens, range(64 + first, 64 + first + tokens), seed=first + tokens))
    check(make(tokens, range(64 + first, 64 + first + tokens), seed=first, scales=(-20, -15)))


@pytest.mark.parametrize("page,block", [(16, 16), (32, 32), (64, 64), (128, 128), (128, 32), (48, 16),
                                        (256, 128)])
@pytest.mark.parametrize("tokens", [1, 60, 300, 2300])
def test_pages_and_blocks(page, block, tokens):
    """(2300 tokens go through the table of slots, the others through a scan)"""
    pages = -(-(tokens + page) // page) + 1
    check(make(tokens, range(page - 5, page - 5 + tokens), page=page, block=block, pages=pages))


@pytest.mark.parametrize("D,rot,pairs", [(128, 128, "half"), (128, 64, "adjacent"), (80, 48, "adjacent"),
                                         (112, 112, "half"), (64, 24, "half"), (72, 20, "half"),
                                         (66, 6, "adjacent"), (16, 16, "half"), (256, 128, "half"),
                                         (512, 256, "half")])
@pytest.mark.parametrize("tokens", [1, 40, 600, 2100])
def test_heads_and_rotations(D, rot, pairs, tokens):
    check(make(tokens, range(7, 7 + tokens), D=D, rot=rot, pairs=pairs, pages=70, dtype=F16))


@pytest.mark.parametrize("heads", [(1, 1), (3, 1), (8, 8), (40, 5), (32, 33), (2, 130)])
@pytest.mark.parametrize("tokens", [1, 50, 520, 2050])
def test_head_counts(heads, tokens):
    check(make(tokens, range(3, 3 + tokens), heads=heads, pages=70, D=32, rot=32))


@pytest.mark.parametrize("tokens", [12, 200, 513, 2000, 2049, 5000])
@pytest.mark.parametrize("slot_type", [torch.int32, torch.int64])
def test_any_order_of_slots(tokens, slot_type):
    """A decode batch, and tokens whose blocks are met in any order, some of them stored nowhere."""
    g = torch.Generator().manual_seed(tokens)
    pages = -(-tokens * 3 // 2 // 32) + 2
    slots = torch.randperm(pages * 32, generator=g)[:tokens]
    slots[::7] = -1
    slots[3] = pages * 32
    slots[4] = -2 ** 31
    check(make(tokens, slots, pages=pages, slot_type=slot_type))


def test_every_slot_nowhere():
    for tokens in (5, 600, 2500):
        check(make(tokens, [-1] * tokens))


@pytest.mark.parametrize("layout", ["nhd", "hnd"])
@pytest.mark.parametrize("axes,sections,order", [(3, (12, 10, 10), "cyclic"), (2, (32, 0), "blocks"),
                                                 (4, (8, 8, 8, 8), "blocks")])
def test_axes_and_layouts(layout, axes, sections, order):
    for tokens in (9, 530, 2100):
        check(make(tokens, range(20, 20 + tokens), axes=axes, sections=sections, order=order, pages=70,
                   layout=layout))


def test_positions_outside_the_table():
    c = make(20, range(20))
    c["positions"][3], c["positions"][4] = 500, -1
    got = call(c)
    assert got["q"][3:5].isnan().all() and (got["k_cache"].view(-1, 2, 64)[3:5] & 0x7f == 0x7f).all()
    check(c)


def test_numbers_at_the_limits():
    """Zeros, infinities, NaN, the smallest and the largest numbers of the type."""
    for dtype, big in ((BF, 2.0 ** 120), (F16, 60000.0)):
        c = make(96, range(96), dtype=dtype, heads=(2, 2), pages=4)
        x = c["qkv"]
        x[0:16, 2:] = 0
        x[16:32, 2:] = 2.0 ** -24 if dtype == F16 else 2.0 ** -120
        x[33, 2:, 5] = math.inf
        x[34, 2:, 6] = -math.inf
        x[50, 2:, 7] = math.nan
        x[64:80, 2:] *= big
        c["positions"][:] = 0  # (turned by nothing: 0 x infinity is met in the sine's products)
        got = call(c)
        codes, scale = append(x[:, 4:].float(), c["v_cache"], c["v_scale"], c["slots"])
        assert torch.equal(got["v_scale"], scale)
        nan = codes & 0x7f == 0x7f
        assert torch.equal(got["v_cache"][~nan], codes[~nan])
        assert (got["v_cache"][nan] & 0x7f == 0x7f).all()
        check(c)


@pytest.mark.parametrize("old", [0.0, -1.0, math.nan, math.inf, 0.3, 1e-30, 1e30, 5.0])
@pytest.mark.parametrize("tokens", [2, 600, 2100])
def test_scales_so_far(old, tokens):
    """Scales that are none start anew, others go up to a power of two within the limits."""
    c = make(tokens, range(5, 5 + tokens), pages=70)
    c["k_scale"][:], c["v_scale"][:] = old, old
    check(c)


def test_nan_codes_stay():
    c = make(1, [17], scales=(-20, -19))
    c["k_cache"][0, 16] = 0x7f
    c["k_cache"][0, 18:] = 0xff  # rows behind the last: left as they are
    check(c)


def test_one_of_two_tokens_with_a_slot_is_kept_whole():
    for tokens in (10, 600, 2100):
        slots = torch.arange(tokens)
        slots[tokens // 2:] = slots[:tokens - tokens // 2].clone()
        c = make(tokens, slots, pages=70)
        got = call(c)
        _, k, v = c["qkv"].split([4, 2, 2], 1)
        k = turned(k, c["positions"], c["table"], "half")
        scale = got["v_scale"].repeat_interleave(16, 1).view(-1, 2)
        held = got["v_cache"].view(FP8).float().view(-1, 2, 64) * scale[..., None]
        for s in range(tokens // 2):
            off = [(held[s] - v[t].float()).abs() <= 2.0 ** -4 * v[t].float().abs()
                   + 2.0 ** -10 * scale[s][:, None] for t in (s, s + tokens // 2)]
            assert off[0].all() or off[1].all()


def test_step_by_step_and_at_once():
    """A prompt token by token: each element within half a step of its own, and of the block's scale."""
    c = make(64, range(64), pages=2, block=32, D=128, rot=128)
    whole = call(c)
    step = dict(c)
    for t in range(64):
        one = dict(step, qkv=c["qkv"][t:t + 1], positions=c["positions"][t:t + 1],
                   slots=c["slots"][t:t + 1])
        step.update({n: x for n, x in call(one).items() if n != "q"})
    assert torch.equal(whole["k_scale"], step["k_scale"])
    assert torch.equal(whole["v_scale"], step["v_scale"])
    for n in ("k", "v"):
        s = whole[n + "_scale"].repeat_interleave(32, 1)[..., None]
        a, b = (x[n + "_cache"].view(FP8).float() * s for x in (whole, step))
        # two roundings of one number: its own (half a step of 2^-3, twice) and below the smallest
        # normal number of the scale half a step of 2^-9 each, as often as the scale grew (8 times: the
        # sizes span 2^6 and the first one may be small)
        assert ((a - b).abs() <= 2.0 ** -3 * a.abs() + 8 * 2.0 ** -10 * s).all()


def test_captured_and_replayed():
    for tokens in (6, 700, 2100):
        c = make(tokens, range(3, 3 + tokens), pages=70)
        dev = {n: c[n].cuda() for n in ("qkv", "positions", "table", "slots", "k_scale", "v_scale")}
        caches = [c[n].cuda() for n in ("k_cache", "v_cache")]
        q, k, v = dev["qkv"].split([4, 2, 2], 1)

        def run():
            return ftb.rope_append(q, k, v, dev["positions"], dev["table"], caches[0].view(FP8),
                                   caches[1].view(FP8), dev["slots"], k_scale=dev["k_scale"],
                                   v_scale=dev["v_scale"])

        run()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run()
        other = make(tokens, range(40, 40 + tokens), pages=70, seed=4)
        for n in dev:
            dev[n].copy_(other[n])
        for a, n in zip(caches, ("k_cache", "v_cache")):
            a.copy_(other[n])
        graph.replay()
        want = call(other)
        assert torch.equal(out.cpu(), want["q"]) and torch.equal(caches[0].cpu(), want["k_cache"])
        assert torch.equal(caches[1].cpu(), want["v_cache"])
        assert torch.equal(dev["k_scale"].cpu(), want["k_scale"])


def test_after_an_attention_on_the_same_stream():
    """The two calls share a workspace: neither minds what the other left."""
    from tests.fp8_cases import Fp8Case, build, reference
    from tests.test_gpu_fp8_attention import compare

    a = Fp8Case([(1, 7000)], cu=False)
    ref = reference(a, *build(a))
    for i in range(3):
        compare(a, *ftb.paged_attention(**a.t, return_lse=True, check_status=True), *ref)
        check(make(2100, range(2100), pages=70, seed=i))


def test_q_in_place():
    c = make(8, range(8))
    dev = c["qkv"].cuda()
    q, k, v = (x.contiguous() for x in dev.split([4, 2, 2], 1))
    want = call(c)["q"]
    kc, vc = c["k_cache"].cuda().view(FP8), c["v_cache"].cuda().view(FP8)
    out = ftb.rope_append(q, k, v, c["positions"].cuda(), c["table"].cuda(), kc, vc, c["slots"].cuda(),
                          k_scale=c["k_scale"].cuda(), v_scale=c["v_scale"].cuda(), q_out=q)
    assert out is q and torch.equal(q.cpu(), want)


def test_offsets_past_32_bits():
    """Caches of more than 2^32 bytes: the last pages are written like the first, found by a scan and by
    the table of slots."""
    page, heads, D = 64, 8, 128
    pages = (1 << 32) // (page * heads * D) + 64
    big = [torch.empty(pages, page, heads, D, dtype=torch.uint8, device="cuda") for _ in "kv"]
    scales = [torch.zeros(pages, 1, heads, device="cuda") for _ in "kv"]
    for tokens in (70, 2200):
        last = -(-tokens // page) + 1
        c = make(tokens, range(3, 3 + tokens), heads=(8, 8), D=D, rot=D, page=page, block=64, pages=last)
        want = call(c)
        far = slice(pages - last, pages)
        for t, n in zip(big, ("k_cache", "v_cache")):
            t[far] = c[n].cuda()
        for t, n in zip(scales, ("k_scale", "v_scale")):
            t[far] = c[n].cuda()
        q, k, v = c["qkv"].cuda().split([8, 8, 8], 1)
        slots = c["slots"].cuda() + (pages - last) * page
        out = ftb.rope_append(q, k, v, c["positions"].cuda(), c["table"].cuda(), big[0].view(FP8),
                              big[1].view(FP8), slots, k_scale=scales[0], v_scale=scales[1])
        assert torch.equal(out.cpu(), want["q"])
        for t, n in zip(big + scales, ("k_cache", "v_cache", "k_scale", "v_scale")):
            assert torch.equal(t[far].cpu(), want[n]), n


def test_calls_of_two_threads_and_two_streams():
    """Threads on one stream, and calls on several streams at once, each with its own caches."""
    import threading

    cases = [make(n, range(5, 5 + n), pages=80, seed=n) for n in (40, 2300, 700, 2500)]
    wants = [call(c) for c in cases]
    errors = []

    def work(c, want, stream):
        try:
            with torch.cuda.stream(stream):
                for _ in range(4):
                    got = call(c)
                    assert all(torch.equal(got[n], want[n]) for n in want)
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    shared = torch.cuda.Stream()
    streams = [shared, shared, torch.cuda.Stream(), torch.cuda.Stream()]
    threads = [threading.Thread(target=work, args=a) for a in zip(cases, wants, streams)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors


def test_captured_before_any_call():
    """A call captured on a stream that has run none has a workspace of its own."""
    c = make(2100, range(9, 2109), pages=80, seed=3)
    dev = {n: c[n].cuda() for n in ("qkv", "positions", "table", "slots", "k_scale", "v_scale", "k_cache",
                                    "v_cache")}
    start = {n: x.clone() for n, x in dev.items()}
    q, k, v = dev["qkv"].split([4, 2, 2], 1)
    stream = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=stream):
        out = ftb.rope_append(q, k, v, dev["positions"], dev["table"], dev["k_cache"].view(FP8),
                              dev["v_cache"].view(FP8), dev["slots"], k_scale=dev["k_scale"],
                              v_scale=dev["v_scale"])
    want = call(c)
    for _ in range(3):
        for n in ("k_cache", "v_cache", "k_scale", "v_scale"):
            dev[n].copy_(start[n])
        graph.replay()
        assert torch.equal(out.cpu(), want["q"])
        for n in ("k_cache", "v_cache", "k_scale", "v_scale"):
            assert torch.equal(dev[n].cpu(), want[n])


def test_refusals():
    c = make(4, range(4))
    q, k, v = c["qkv"].cuda().split([4, 2, 2], 1)
    good = dict(k_cache=c["k_cache"].cuda().view(FP8), v_cache=c["v_cache"].cuda().view(FP8),
                slots=c["slots"].cuda(), k_scale=c["k_scale"].cuda(), v_scale=c["v_scale"].cuda())
    pos, table = c["positions"].cuda(), c["table"].cuda()
    ftb.rope_append(q, k, v, pos, table, **good)
    for bad in (dict(k_scale=None), dict(v_scale=None), dict(k_cache=good["k_cache"].view(torch.uint8)),
                dict(k_cache=good["k_cache"].view(torch.uint8).bfloat16()), dict(slots=None),
                dict(k_scale=good["k_scale"].half()), dict(v_scale=good["v_scale"][:, :1]),
                dict(k_scale=good["k_scale"].cpu()), dict(slots=good["slots"][:3]),
                dict(k_scale=good["k_scale"][:, :, :1], v_scale=good["v_scale"][:, :, :1]),
                dict(v_cache=good["v_cache"][:, :16])):
        with pytest.raises(ValueError):
            ftb.rope_append(q, k, v, pos, table, **{**good, **bad})
    # (the caches are held in 8 bits, so a call without scales is refused too)
    with pytest.raises(ValueError):
        ftb.rope_append(q, k, v, pos, table, good["k_cache"], good["v_cache"], good["slots"])
