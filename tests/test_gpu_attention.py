"""ftb.paged_attention against the definition in 64 bits (tests/attn_cases.py has the bounds).
Every cache row that no token may see holds NaN (or infinity), and unused block-table entries
name no page."""
import math

import pytest
import torch

import ftb
from tests.attn_cases import AttnCase, build, reference

pytestmark = pytest.mark.gpu
BF, F16 = torch.bfloat16, torch.float16


def check(c: AttnCase):
    q, keys = build(c)
    out, lse = ftb.paged_attention(**c.t, window=c.window, causal=c.causal, scale=c.scale,
                                   return_lse=True, check_status=True)
    ref, bound, ref_lse = reference(c, q, keys)
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
    check(AttnCase([(1, kv)], dtype=dtype, cu=False, seed=kv))


@pytest.mark.parametrize("page", [8, 16, 32, 64, 128, 256])
@pytest.mark.parametrize("head", [8, 64, 72, 80, 112, 128])
def test_one_token_pages_and_heads(page, head):
    check(AttnCase([(1, 300), (1, 1), (1, 0), (1, 513)], page=page, head=head, cu=False))


@pytest.mark.parametrize("heads", [(1, 1), (5, 1), (7, 7), (16, 1), (24, 8), (32, 4), (17, 1),
                                   (64, 1), (128, 1)])
def test_head_groups(heads):
    check(AttnCase([(1, 70), (1, 333)], q_heads=heads[0], kv_heads=heads[1], cu=False))


def test_decode_batch_larger_than_the_block():
    check(AttnCase([(1, (37 * i) % 260) for i in range(401)], q_heads=4, kv_heads=2, head=64,
                   cu=False))


def test_decode_long_split_over_blocks():
    check(AttnCase([(1, 20011), (1, 3), (1, 9000)], q_heads=8, kv_heads=2, page=64, cu=False))


@pytest.mark.parametrize("window", [1, 7, 64, 65, 500])
def test_one_token_window(window):
    check(AttnCase([(1, 700), (1, 64), (1, 5)], window=window, cu=False))


# ---- chunks of new tokens ----
@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("pairs", [[(1, 1)], [(2, 2)], [(5, 5)], [(33, 33)], [(128, 128)],
                                   [(129, 200)], [(300, 1000)], [(64, 64), (65, 65), (1, 900)]])
def test_chunk(pairs, dtype):
    check(AttnCase(pairs, dtype=dtype))


@pytest.mark.parametrize("page", [8, 16, 64, 128, 256])
@pytest.mark.parametrize("head", [8, 64, 80, 112, 128])
def test_chunk_pages_and_heads(page, head):
    check(AttnCase([(150, 410), (0, 90), (3, 3)], page=page, head=head))


@pytest.mark.parametrize("heads", [(1, 1), (3, 1), (5, 1), (12, 4), (7, 1), (8, 8), (32, 2),
                                   (48, 1), (128, 1)])
def test_chunk_head_groups(heads):
    check(AttnCase([(77, 190), (20, 20)], q_heads=heads[0], kv_heads=heads[1], head=64))


@pytest.mark.parametrize("window", [1, 16, 100, 128, 129, 1000])
def test_chunk_window(window):
    check(AttnCase([(200, 600), (40, 40), (1, 333)], window=window))


def test_chunk_not_causal():
    check(AttnCase([(130, 300), (17, 17), (1, 9)], causal=False))
    check(AttnCase([(130, 300), (17, 17)], causal=False, window=50))


def test_rows_without_keys():
    # more new tokens than keys: the first ones precede every key
    check(AttnCase([(40, 10), (3, 0), (200, 150), (1, 0)]))
    check(AttnCase([(1, 0), (1, 0)], cu=False))


@pytest.mark.parametrize("pairs", [[(1, 200)] * 3, [(150, 260), (9, 9)]])
def test_layouts_and_strides(pairs):
    check(AttnCase(pairs, layout="hnd", q_slice=True, page=32))
    check(AttnCase(pairs, layout="hnd", q_slice=True, head=72, page=16, dtype=F16))


@pytest.mark.parametrize("pairs", [[(1, 300)], [(140, 300)]])
def test_infinity_in_unused_rows(pairs):
    check(AttnCase(pairs, poison=math.inf))
    check(AttnCase(pairs, poison=-math.inf, dtype=F16, window=90))


@pytest.mark.parametrize("pairs", [[(1, 900)], [(150, 900)]])
@pytest.mark.parametrize("scale", [-0.09, 0.0, 0.5])
def test_scales(pairs, scale):
    """A negative scale, a flat softmax and a sharp one (scores up to 2^4 times 4)."""
    check(AttnCase(pairs, scale=scale))


@pytest.mark.parametrize("pairs", [[(1, 400)], [(140, 400)]])
def test_rising_scores_move_the_maximum(pairs):
    """Each key scores higher than the last, by far more than the accumulators' headroom."""
    c = AttnCase(pairs, q_heads=2, kv_heads=1, head=64, causal=False, scale=1.0)
    q, keys = build(c)
    n, kv = pairs[0]
    c.t["q"].zero_()
    c.t["q"][..., 0] = 1.0
    ramp = torch.arange(kv, dtype=torch.float32) * 0.5 - 60.0
    table, page = c.t["block_table"][0].long(), c.page
    flat = c.t["k_cache"][table[:-(-kv // page)]]
    rows = flat.view(-1, 1, 64)
    rows[:kv] = 0
    rows[:kv, 0, 0] = ramp.to(BF).to("cuda")
    c.t["k_cache"][table[:-(-kv // page)]] = flat
    x = keys[0].clone()
    x[:, 0] = 0
    x[:, 0, 0, 0] = ramp.to(BF)
    qr = torch.zeros_like(q)
    qr[..., 0] = 1.0
    out, lse = ftb.paged_attention(**c.t, causal=False, scale=1.0, return_lse=True)
    ref, bound, ref_lse = reference(c, qr, [x])
    # scores reach 2^7: fp32 rounds them at 2^-17, within the exponential's 2^-14
    assert ((out.double().cpu() - ref).abs() <= bound).all()
    assert (lse.double().cpu() - ref_lse).abs().max() <= 2.0 ** -13


def test_splits_do_not_change_with_order_of_arrival():
    c = AttnCase([(1, 30000), (1, 12345)], q_heads=8, kv_heads=1, page=64, cu=False)
    build(c)
    first = ftb.paged_attention(**c.t).clone()
    for _ in range(20):
        assert torch.equal(ftb.paged_attention(**c.t), first)
    c = AttnCase([(60, 5000)], q_heads=8, kv_heads=1, page=64)
    build(c)
    first = ftb.paged_attention(**c.t).clone()
    for _ in range(20):
        assert torch.equal(ftb.paged_attention(**c.t), first)


def test_offsets_past_32_bits():
    """Cache rows past 2^32 bytes and 2^31 elements from the cache's start."""
    page, heads, head = 64, 8, 128
    pages = (2 ** 31) // (page * heads * head) + 40
    k = torch.zeros(pages, page, heads, head, dtype=BF, device="cuda")
    v = torch.zeros_like(k)
    g = torch.Generator(device="cuda").manual_seed(3)
    k[-4:].normal_(generator=g)
    v[-4:].normal_(generator=g)
    for n, total in ((1, 200), (130, 200)):
        q = torch.randn(n, 8, head, generator=g, device="cuda").to(BF)
        args = dict(kv_len=torch.tensor([total], dtype=torch.int32, device="cuda"),
                    cu_q=torch.tensor([0, n], dtype=torch.int32, device="cuda"), max_q=n)
        table = torch.arange(pages - 4, pages, dtype=torch.int32, device="cuda")[None]
        far = ftb.paged_attention(q, k, v, table, **args, check_status=True)
        near = ftb.paged_attention(q, k[-4:].clone(), v[-4:].clone(), table - (pages - 4), **args)
        assert torch.equal(far, near) and far.abs().max() > 0


@pytest.mark.parametrize("pairs,cu", [([(1, 500), (1, 77)], False), ([(90, 400)], True)])
def test_status_word(pairs, cu):
    def call(c, **kw):
        return ftb.paged_attention(**{**c.t, **kw}, check_status=True)

    c = AttnCase(pairs, cu=cu)
    build(c)
    good = call(c)
    bad = c.t["block_table"].clone()
    bad[0, 1] = 10 ** 6  # no such page
    with pytest.raises(ValueError, match="status 1"):
        call(c, block_table=bad)
    with pytest.raises(ValueError, match="status 1"):
        call(c, kv_len=c.t["kv_len"] + 10 ** 6)
    if cu:
        with pytest.raises(ValueError, match="status 2"):
            call(c, cu_q=torch.tensor([0, 91], dtype=torch.int32, device="cuda"))
        with pytest.raises(ValueError, match="status 2"):
            call(c, max_q=89)
    assert torch.equal(call(c), good)  # and nothing stays behind


def test_another_stream_and_a_graph():
    c = AttnCase([(1, 3000), (1, 50)], cu=False)
    build(c)
    want = ftb.paged_attention(**c.t).clone()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = ftb.paged_attention(**c.t)
    s.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    out = torch.empty_like(want)
    with torch.cuda.stream(s):
        ftb.paged_attention(**c.t, out=out)
        s.synchronize()
        with torch.cuda.graph(graph, stream=s):
            ftb.paged_attention(**c.t, out=out)
    out.zero_()
    c.t["kv_len"].copy_(torch.tensor([2900, 50], dtype=torch.int32))  # lengths are read on replay
    graph.replay()
    torch.cuda.synchronize()
    again = ftb.paged_attention(**c.t)
    assert torch.equal(out, again) and not torch.equal(out, want)


@pytest.mark.parametrize("c", [
    AttnCase([(700, 1700)], q_heads=64, kv_heads=1, head=64),  # 175 items, a few more than blocks
    AttnCase([(700, 1700)], q_heads=64, kv_heads=1, head=64, window=1100),
    AttnCase([(256, 2300)], q_heads=160, kv_heads=160, head=8),  # more heads than parts' room
], ids=["left", "left-window", "heads"])
def test_items_left_over_after_whole_rounds(c):
    check(c)


def attend(c, **kw):
    return ftb.paged_attention(**{**c.t, **kw})


def test_a_graph_without_an_eager_call_and_a_grown_workspace():
    """The capture makes its own workspace, zeroed at each replay; a workspace that a graph holds
    stays when a larger call replaces it."""
    small = AttnCase([(1, 3000), (1, 50)], cu=False)
    large = AttnCase([(300, 700), (90, 90), (2, 3000)])
    build(small), build(large)
    want, want_large = attend(small).clone(), attend(large).clone()
    for eager_first in (False, True):
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        graph, out = torch.cuda.CUDAGraph(), torch.empty_like(want)
        with torch.cuda.stream(s):
            if eager_first:
                ftb.paged_attention(**small.t, out=out)
                s.synchronize()
            with torch.cuda.graph(graph, stream=s):
                ftb.paged_attention(**small.t, out=out)
            for _ in range(2):
                assert torch.equal(ftb.paged_attention(**large.t), want_large)
                out.zero_()
                graph.replay()
                s.synchronize()
                assert torch.equal(out, want)


@pytest.mark.parametrize("pairs", [[(5, 70), (0, 9), (3, 3)], [(400, 900), (0, 9), (129, 129)]])
def test_a_loose_max_q_and_rows_of_no_sequence(pairs):
    """max_q may be any bound (a model's longest), and rows behind the last sequence stay."""
    c = AttnCase(pairs)
    build(c)
    want = attend(c)
    assert torch.equal(attend(c, max_q=1 << 20), want)
    q = torch.cat([c.t["q"], torch.full_like(c.t["q"][:7], math.nan)])
    out = torch.full_like(q, 3.0)
    attend(c, q=q, out=out)
    assert torch.equal(out[:-7], want) and (out[-7:] == 3.0).all()


def test_refusals():
    c = AttnCase([(1, 50), (1, 60)], cu=False)
    build(c)

    def refuse(match=None, **kw):
        with pytest.raises((ValueError, ftb._lib.FtbError), match=match):
            ftb.paged_attention(**{**c.t, **kw})

    t = c.t
    refuse(q=t["q"].float())
    refuse(q=t["q"][:1])
    refuse(q=t["q"].half())
    refuse(q=t["q"][:, :3])  # 3 query heads over 2 kv heads
    refuse(k_cache=t["k_cache"][..., :64])
    refuse(k_cache=t["k_cache"][:, :12], v_cache=t["v_cache"][:, :12])  # page of 12
    refuse(block_table=t["block_table"].long())
    refuse(block_table=t["block_table"][:1])
    refuse(kv_len=t["kv_len"].long())
    refuse(window=-1)
    refuse(max_q=2)
    refuse(scale=float("nan"))
    refuse(cu_q=t["kv_len"])
    refuse(out=torch.empty(2, 8, 128, device="cuda"))
    refuse(block_table=t["block_table"].cpu())
    refuse(q=t["q"].cpu())


def test_empty_calls():
    c = AttnCase([(1, 50)], cu=False)
    build(c)
    out = ftb.paged_attention(c.t["q"][:0], c.t["k_cache"], c.t["v_cache"],
                              c.t["block_table"][:0], c.t["kv_len"][:0])
    assert out.shape == (0, 8, 128)
