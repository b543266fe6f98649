"""ftb.paged_attention where a row's scores all lie far below zero: softmax does not change under a
shift of all scores, so the output has to be right wherever they lie.

Bounds, beside those of tests/attn_cases.py: the shift is one product of about 2^11 before the
scale of 2^-3.5, so each of the up to 128 products of a score may be cut to that sum's last place,
2^-12: 2^-5 in all, 2^-8.5 after the scale. A weight is off by that on both sides of the division:
2^-7.5 < 2^-7 of A. lse: 2^-8.5, and the rounding of its own 2^8 many times smaller: 2^-8."""
import math

import pytest
import torch

import ftb
from tests.attn_cases import U, AttnCase, build, reference

pytestmark = pytest.mark.gpu
BF, F16 = torch.bfloat16, torch.float16


def rewrite_keys(c, keys):
    """Writes keys[b][:, 0] to the cache rows that some token may see."""
    table, page = c.t["block_table"].cpu().long(), c.page
    for b, ((n, kv), x) in enumerate(zip(c.pairs, keys)):
        j = torch.arange(max(0, kv - n - c.window + 1) if c.window else 0, kv)
        c.t["k_cache"][table[b, j // page].cuda(), (j % page).cuda()] = x[j, 0].cuda()


def shifted(c, by):
    """The case's inputs with `by` added to every score: one constant component of q and of k."""
    q, keys = build(c)
    q, keys = q.clone(), [x.clone() for x in keys]
    q[..., 0] = 32.0
    c.t["q"][..., 0] = 32.0
    for x in keys:
        x[:, 0, :, 0] = by / (32.0 * c.head ** -0.5)
    rewrite_keys(c, keys)
    return q, keys


def check(c, by):
    q, keys = shifted(c, by)
    out, lse = ftb.paged_attention(**c.t, window=c.window, causal=c.causal, return_lse=True,
                                   check_status=True)
    ref, bound, ref_lse = reference(c, q, keys)
    total, _, _ = reference(c, q, [torch.stack([x[:, 0], x[:, 1].abs()], 1) for x in keys])
    out, lse = out.double().cpu(), lse.double().cpu()
    assert torch.isfinite(out).all()
    seen = torch.isfinite(ref_lse)
    assert torch.equal(torch.isfinite(lse), seen)
    assert ((lse - ref_lse)[seen].abs() <= 2.0 ** -8).all()
    worst = ((out - ref).abs() / (bound + 2.0 ** -7 * total)).max().item()
    assert worst <= 1.0, f"out off by {worst} of its bound"


@pytest.mark.parametrize("by", [-85.0, -100.0, -200.0])
@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("c", [
    dict(pairs=[(64, 1025)], q_heads=32, kv_heads=8, page=64),
    dict(pairs=[(256, 1000)], q_heads=32, kv_heads=8, page=64),
    dict(pairs=[(256, 5000)], q_heads=16, kv_heads=16, window=1000, page=32),
    dict(pairs=[(256, 1000)], q_heads=32, kv_heads=8, page=64, causal=False),
    dict(pairs=[(700, 1700)], q_heads=16, kv_heads=16, page=64),
    dict(pairs=[(1, 9000), (1, 1)], cu=False, page=64),
    dict(pairs=[(9, 3000), (3, 3)], q_heads=4, kv_heads=4, window=70),
], ids=["last-part", "parts", "window", "not-causal", "whole", "decode", "few-rows"])
def test_low_scores(c, dtype, by):
    """Cut items have parts in which some rows see no key."""
    check(AttnCase(**c, dtype=dtype), by)



def test_f16_weights_under_a_low_maximum():
    """One key at a score of -5 and 16383 12.5 below it, which hold 6 % of the sum together: in
    f16 a weight is good to 2^-25 of the largest where the reference is not above it, so 2^-25
    times the number of keys over the sum comes to the bounds of tests/attn_cases.py, which are
    without their 2^-17 here. Scores are one product each, and exact."""
    heads = torch.cuda.get_device_properties(0).multi_processor_count  # an item per SM, uncut
    c = AttnCase([(17, 16384)], q_heads=heads, kv_heads=heads, head=8, page=64, dtype=F16,
                 causal=False, scale=1.0)
    _, keys = build(c)
    x = torch.zeros_like(keys[0])
    x[:, 0, :, 0] = -17.5
    x[:, 1] = 1.0
    x[7, 0, :, 0], x[7, 1] = -5.0, -1.0
    rewrite_keys(c, [x])
    c.t["v_cache"].fill_(1.0)
    page = int(c.t["block_table"][0, 0])
    c.t["v_cache"][page, 7] = -1.0
    c.t["q"].zero_()
    c.t["q"][..., 0] = 1.0
    out, lse = ftb.paged_attention(**c.t, causal=False, scale=1.0, return_lse=True)
    few = 16383 * math.exp(-12.5)
    want, u = (few - 1.0) / (few + 1.0), U[F16]
    bound = u * (abs(want) + 1.0) + 2.0 ** -13 + 2.0 ** -25 * 16384 / (few + 1.0)
    assert (out.double().cpu() - want).abs().max() <= bound
    assert (lse.double().cpu() - (-5.0 + math.log1p(few))).abs().max() <= 2.0 ** -14
