"""ftb.paged_attention over an 8-bit cache against the definition in 64 bits (tests/fp8_cases.py has the
bounds). Every row and scale that no token may see holds NaN or infinity, and unused block-table entries
name no page."""
import math

import pytest
import torch

import ftb
from tests.fp8_cases import FP8, Fp8Case, build, reference

pytestmark = pytest.mark.gpu
BF, F16 = torch.bfloat16, torch.float16


def check(c: Fp8Case):
    q, keys = build(c)
    out, lse = ftb.paged_attention(**c.t, window=c.window, causal=c.causal, scale=c.scale,
                                   return_lse=True, check_status=True)
    compare(c, out, lse, *reference(c, q, keys))


def compare(c, out, lse, ref, bound, ref_lse):
    out, lse = out.double().cpu(), lse.double().cpu()
    assert torch.isfinite(out).all()
    worst = ((out - ref).abs() / bound).max().item() if out.numel() else 0.0
    assert worst <= 1.0, f"out off by {worst} of its bound"
    empty = torch.isinf(ref_lse)
    assert torch.equal(lse[empty], ref_lse[empty])
    assert (out[empty] == 0).all()
    d = (lse - ref_lse)[~empty].abs()
    assert (d <= 2.0 ** -14 + 2.0 ** -21 * ref_lse[~empty].abs()).all(), d.max()


# ---- one new token per sequence ----
@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("kv", [1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 1000])
def test_one_token(kv, dtype):
    check(Fp8Case([(1, kv)], dtype=dtype, cu=False, seed=kv))


@pytest.mark.parametrize("page,block", [(16, 16), (32, 16), (32, 32), (64, 16), (64, 64), (128, 32),
                                        (128, 128), (256, 64), (256, 128), (512, 16)])
@pytest.mark.parametrize("head", [16, 64, 80, 112, 128])
def test_one_token_pages_and_heads(page, block, head):
    check(Fp8Case([(1, 300), (1, 1), (1, 0), (1, 513)], page=page, block=block, head=head, cu=False))


@pytest.mark.parametrize("heads", [(1, 1), (5, 1), (7, 7), (16, 1), (24, 8), (32, 4), (17, 1),
                                   (64, 1), (128, 1)])
def test_head_groups(heads):
    check(Fp8Case([(1, 70), (1, 333)], q_heads=heads[0], kv_heads=heads[1], cu=False))


def test_decode_batch_larger_than_the_block():
    check(Fp8Case([(1, (37 * i) % 260) for i in range(401)], q_heads=4, kv_heads=2, head=64,
                  cu=False))


def test_decode_long_split_over_blocks():
    check(Fp8Case([(1, 20011), (1, 3), (1, 9000)], q_heads=8, kv_heads=2, page=64, block=32, cu=False))


@pytest.mark.parametrize("kv_heads", [1, 2, 3, 6, 8])
@pytest.mark.parametrize("head", [64, 80, 128])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
def test_decode_batch_by_one_head_and_by_pairs(page, head, kv_heads):
    """Enough keys for two heads at a time (even numbers of kv heads), in any pages, with sequences
    without keys, windows over parts of tiles and rows beyond one token."""
    g = torch.Generator().manual_seed(page + head + kv_heads)
    kv = torch.randint(0, 700, (90,), generator=g).tolist()
    c = Fp8Case([(1, n) for n in kv], q_heads=4 * kv_heads, kv_heads=kv_heads, head=head, page=page,
                cu=False, window=333 if page == 32 else 0, dtype=F16 if page == 64 else BF)
    check(c)
    check(Fp8Case([(2, n) for n in kv[:60]], q_heads=3 * kv_heads, kv_heads=kv_heads, head=head, page=page,
                  block=16))


@pytest.mark.parametrize("window", [1, 7, 64, 65, 500])
def test_one_token_window(window):
    check(Fp8Case([(1, 700), (1, 64), (1, 5)], window=window, cu=False))


# ---- chunks of new tokens ----
@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("pairs", [[(1, 1)], [(2, 2)], [(5, 5)], [(33, 33)], [(128, 128)],
                                   [(129, 200)], [(300, 1000)], [(64, 64), (65, 65), (1, 900)],
                                   [(700, 2100)]])
def test_chunk(pairs, dtype):
    check(Fp8Case(pairs, dtype=dtype))


LARGE = [(600, 1500), (0, 90), (3, 3), (260, 400)]  # more work than the kernel for few rows takes


@pytest.mark.parametrize("page,block", [(16, 16), (32, 32), (64, 16), (64, 64), (128, 128), (256, 32)])
@pytest.mark.parametrize("head", [16, 64, 80, 128])
def test_chunk_pages_and_heads(page, block, head):
    check(Fp8Case([(150, 410), (0, 90), (3, 3)], page=page, block=block, head=head))
    check(Fp8Case(LARGE, page=page, block=block, head=head))


@pytest.mark.parametrize("heads", [(1, 1), (3, 1), (5, 1), (12, 4), (7, 1), (8, 8), (32, 2),
                                   (48, 1), (128, 1)])
def test_chunk_head_groups(heads):
    check(Fp8Case([(77, 190), (20, 20)], q_heads=heads[0], kv_heads=heads[1], head=64))
    check(Fp8Case([(400, 2300)], q_heads=heads[0], kv_heads=heads[1]))


@pytest.mark.parametrize("head", [64, 128])
@pytest.mark.parametrize("dtype", [BF, F16])
def test_more_items_than_multiprocessors(dtype, head):
    """A block takes several items one after another: with keys for both row tiles, for one of them
    (windows, ends of sequences) and for none, of one key tile and of many; rows of q that f16 holds and
    rows that are scaled."""
    pairs = [(300, 2900), (58, 1860), (3, 1200), (260, 1500), (1, 0), (280, 280), (19, 2100), (400, 300)]
    c = Fp8Case(pairs * 3, q_heads=24, kv_heads=8, head=head, page=32, block=32, dtype=dtype, window=900)
    q, keys = build(c)
    if dtype == BF:
        lift = torch.ones(q.shape[:2] + (1,))
        lift[::3, ::2] = 2.0 ** -12
        q = (q.float() * lift).to(BF)
        c.t["q"] = q.cuda()
    for _ in range(20):
        out, lse = ftb.paged_attention(**c.t, window=c.window, return_lse=True, check_status=True)
    compare(c, out, lse, *reference(c, q, keys))


@pytest.mark.parametrize("window", [1, 16, 100, 128, 129, 1000])
def test_chunk_window(window):
    check(Fp8Case([(200, 600), (40, 40), (1, 333)], window=window))
    check(Fp8Case([(900, 2000), (40, 40), (1, 333)], window=window, q_heads=16, page=32, block=32))


def test_chunk_not_causal():
    check(Fp8Case([(130, 300), (17, 17), (1, 9)], causal=False))
    check(Fp8Case([(700, 1300), (17, 17)], causal=False, window=50, q_heads=16))


def test_rows_without_keys():
    # more new tokens than keys: the first ones precede every key
    check(Fp8Case([(40, 10), (3, 0), (200, 150), (1, 0)]))
    check(Fp8Case([(1500, 1100), (3, 0), (1, 0)], q_heads=16))
    check(Fp8Case([(1, 0), (1, 0)], cu=False))


@pytest.mark.parametrize("pairs", [[(1, 200)] * 3, [(150, 260), (9, 9)], LARGE])
def test_layouts_and_strides(pairs):
    check(Fp8Case(pairs, layout="hnd", q_slice=True, page=32))
    check(Fp8Case(pairs, layout="hnd", q_slice=True, head=80, page=64, block=32, dtype=F16))


@pytest.mark.parametrize("pairs", [[(1, 900)], [(150, 900)], [(800, 900)]])
@pytest.mark.parametrize("scale", [-0.09, 0.0, 0.5])
def test_softmax_scales(pairs, scale):
    check(Fp8Case(pairs, scale=scale, q_heads=16, spread=0.5))


# ---- scales of blocks ----
@pytest.mark.parametrize("pairs", [[(1, 900), (1, 40)], [(150, 900)], [(700, 1500)]])
@pytest.mark.parametrize("dtype", [BF, F16])
def test_scales_that_are_no_powers_of_two(pairs, dtype):
    check(Fp8Case(pairs, dtype=dtype, odd_scales=True, page=64, block=32))


@pytest.mark.parametrize("pairs", [[(1, 900), (1, 40)], [(150, 900)], [(700, 1500)]])
def test_value_scales_far_apart(pairs):
    """Blocks whose V differ by up to 2^60: no weight is lost beside its block's scale."""
    c = Fp8Case(pairs, page=64, block=16, q_heads=16)
    q, keys = build(c)
    g = torch.Generator().manual_seed(3)
    s = c.t["v_scale"]
    e = torch.randint(-30, 31, s.shape, generator=g).float().exp2().cuda()
    c.t["v_scale"] = torch.where(s.isnan(), s, e)
    table = c.t["block_table"].cpu()
    for b, (_, kv) in enumerate(pairs):
        j = torch.arange(kv)
        vs = c.t["v_scale"].cpu()[table[b].long()[j // 64], j % 64 // 16].double()
        keys[b][1] = (keys[b][1][0], vs)
    out, lse = ftb.paged_attention(**c.t, return_lse=True, check_status=True)
    compare(c, out, lse, *reference(c, q, keys))


def test_scales_outside_the_limits_are_the_limits():
    c = Fp8Case([(1, 64)], page=64, block=16, cu=False)
    build(c)
    low = {**c.t, "k_scale": torch.full_like(c.t["k_scale"], 2.0 ** -40),
           "v_scale": torch.full_like(c.t["v_scale"], 2.0 ** 40)}
    odd = {**c.t, "k_scale": torch.full_like(c.t["k_scale"], math.nan),
           "v_scale": torch.full_like(c.t["v_scale"], math.inf)}
    odd["k_scale"][:, 1], odd["k_scale"][:, 2] = 0.0, -3.0
    assert torch.equal(ftb.paged_attention(**low), ftb.paged_attention(**odd))


# ---- q beyond f16 ----
@pytest.mark.parametrize("pairs", [[(1, 300)], [(100, 300)], [(700, 1500)]])
@pytest.mark.parametrize("power", [-90, -20, 30])
def test_bf16_queries_of_any_size(pairs, power):
    """Every other head's q times 2^power, the softmax's scale times 2^-power or so."""
    c = Fp8Case(pairs, page=64, block=64, q_heads=16, scale=128 ** -0.5 * 2.0 ** -max(power, -30))
    q, keys = build(c)
    lift = torch.ones(q.shape[:2] + (1,))
    lift[:, ::2] = 2.0 ** power
    if power < 0:  # (the other heads' scores stay small too)
        lift[:, 1::2] = 2.0 ** -25
    q = (q.float() * lift).to(BF)
    c.t["q"] = q.cuda()
    out, lse = ftb.paged_attention(**c.t, scale=c.scale, return_lse=True, check_status=True)
    compare(c, out, lse, *reference(c, q, keys))


@pytest.mark.parametrize("pairs", [[(1, 300)], [(700, 1500)]])
def test_a_large_row_leaves_the_others_alone(pairs):
    c = Fp8Case(pairs, page=64, block=64, q_heads=16)
    q, keys = build(c)
    plain = ftb.paged_attention(**c.t)
    c.t["q"] = c.t["q"].clone()
    c.t["q"][:, ::2] *= 2.0 ** 100
    out = ftb.paged_attention(**c.t)
    assert torch.isfinite(out).all() and torch.equal(out[:, 1::2], plain[:, 1::2])


def test_infinite_and_nan_queries_stay_in_their_rows():
    for pairs in ([(1, 200), (1, 90)], [(700, 1500), (90, 90)]):
        c = Fp8Case(pairs, q_heads=16)
        build(c)
        good = ftb.paged_attention(**c.t)
        c.t["q"][0, 3], c.t["q"][-1, 0, 5] = math.inf, math.nan
        out = ftb.paged_attention(**c.t)
        assert out[0, 3].isnan().all() and out[-1, 0].isnan().all()
        same = torch.ones(out.shape[:2], dtype=torch.bool)
        same[0, 3] = same[-1, 0] = False
        assert torch.equal(out[same], good[same])


# ---- calls ----
def test_captured_on_other_lengths():
    """A captured decode step follows the lengths, the table and the scales it finds at replay."""
    a = Fp8Case([(1, 400), (1, 37), (1, 0)], cu=False, page=32, block=32)
    qa, ka = build(a)
    ftb.paged_attention(**a.t, return_lse=True)
    out, lse = None, None
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = ftb.paged_attention(**a.t, return_lse=True)
    graph.replay()
    compare(a, out, lse, *reference(a, qa, ka))
    b = Fp8Case([(1, 64), (1, 300), (1, 5)], cu=False, page=32, block=32, seed=9)
    qb, kb = build(b)
    for name in ("q", "kv_len"):
        a.t[name].copy_(b.t[name])
    width = min(a.t["block_table"].shape[1], b.t["block_table"].shape[1])
    a.t["block_table"][:, :width] = b.t["block_table"][:, :width]
    for name in ("k_cache", "v_cache", "k_scale", "v_scale"):
        n = b.t[name].shape[0]
        view = torch.uint8 if "cache" in name else torch.float32
        assert n <= a.t[name].shape[0]
        a.t[name].view(view)[:n] = b.t[name].view(view)
    graph.replay()
    compare(b, out, lse, *reference(b, qb, kb))


def test_two_calls_on_two_streams():
    cases = [Fp8Case([(1, 5000)] * 3, cu=False, seed=1), Fp8Case([(700, 2000)], q_heads=16, seed=2)]
    refs = [reference(c, *build(c)) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    outs = []
    for _ in range(3):
        for c, s in zip(cases, streams):
            with torch.cuda.stream(s):
                outs.append(ftb.paged_attention(**c.t, return_lse=True))
    torch.cuda.synchronize()
    for i, (out, lse) in enumerate(outs):
        compare(cases[i % 2], out, lse, *refs[i % 2])


def test_same_bits_every_time():
    for c in (Fp8Case([(1, 9000), (1, 77)], cu=False), Fp8Case([(700, 3000)], q_heads=16)):
        build(c)
        first = ftb.paged_attention(**c.t)
        assert all(torch.equal(first, ftb.paged_attention(**c.t)) for _ in range(5))


def test_rows_of_no_sequence_stay():
    c = Fp8Case([(3, 40), (5, 9)])
    build(c)
    c.t["q"] = torch.cat([c.t["q"], c.t["q"][:4]])
    out = torch.full_like(c.t["q"], 7.0)
    ftb.paged_attention(**c.t, out=out)
    assert (out[8:] == 7).all() and not (out[:8] == 7).all()


def test_bad_pages_are_reported():
    c = Fp8Case([(1, 100)], cu=False)
    build(c)
    c.t["block_table"][0, 2] = c.t["k_cache"].shape[0]
    with pytest.raises(ValueError, match="status 1"):
        ftb.paged_attention(**c.t, check_status=True)
    build(c)
    ftb.paged_attention(**c.t, check_status=True)


def test_offsets_past_32_bits():
    """A cache of more than 2^32 bytes: the last pages are read like the first."""
    page, heads, D = 64, 8, 128
    pages = (1 << 32) // (page * heads * D) + 64
    k = torch.zeros(pages, page, heads, D, dtype=torch.uint8, device="cuda").view(FP8)
    v = torch.zeros(pages, page, heads, D, dtype=torch.uint8, device="cuda").view(FP8)
    ks, vs = (torch.ones(pages, 1, heads, device="cuda") for _ in "kv")
    c = Fp8Case([(1, 200)], q_heads=16, kv_heads=heads, page=page, block=64, cu=False)
    q, keys = build(c)
    ref = reference(c, q, keys)
    ids = c.t["block_table"][0, :4].long()
    far = torch.arange(pages - 4, pages, device="cuda")
    for big, name in ((k, "k_cache"), (v, "v_cache")):
        big.view(torch.uint8)[far] = c.t[name].view(torch.uint8)[ids]
    ks[far], vs[far] = c.t["k_scale"][ids], c.t["v_scale"][ids]
    t = dict(c.t, k_cache=k, v_cache=v, k_scale=ks, v_scale=vs)
    t["block_table"] = t["block_table"].clone()
    t["block_table"][0, :4] = far.int()
    compare(c, *ftb.paged_attention(**t, return_lse=True, check_status=True), *ref)


def test_refusals():
    c = Fp8Case([(1, 100)], cu=False, page=32, block=16)
    build(c)
    ftb.paged_attention(**c.t)
    for bad in (dict(k_scale=None), dict(v_scale=None), dict(k_cache=c.t["k_cache"].view(torch.uint8)),
                dict(k_scale=c.t["k_scale"].double(), v_scale=c.t["v_scale"].double()),
                dict(v_scale=c.t["v_scale"][:, :1]), dict(k_scale=c.t["k_scale"].cpu()),
                dict(q=c.t["q"].float()), dict(q=c.t["q"][..., :64])):
        with pytest.raises(ValueError):
            ftb.paged_attention(**{**c.t, **bad})
    with pytest.raises(ValueError):  # an 8-bit cache without its scales
        ftb.paged_attention(**{**c.t, "k_scale": None, "v_scale": None})


def test_calls_of_two_threads():
    import threading

    cases = [Fp8Case([(1, 4000)] * 9, cu=False, page=64, block=64, seed=1),
             Fp8Case([(600, 1500)], q_heads=16, seed=2)]
    refs = [reference(c, *build(c)) for c in cases]
    errors = []

    def work(i):
        try:
            for _ in range(10):
                compare(cases[i], *ftb.paged_attention(**cases[i].t, return_lse=True), *refs[i])
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in (0, 1, 0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
