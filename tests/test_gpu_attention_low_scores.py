"""ftb.paged_attention where a row's scores all lie far below zero: softmax does not change under a
shift of all scores, so the output has to be right wherever they lie.

Bounds, beside those of tests/attn_cases.py: the shift is one product of about 2^11 before the
scale of 2^-3.5, so each of the up to 128 products of a score may be cut to that sum's last place,
2^-12: 2^-5 in all, 2^-8.5 after the scale. A weight is off by that on both sides of the division:
2^-7.5 < 2^-7 of A. lse: 2^-8.5, and the rounding of its own 2^8 many times smaller: 2^-8."""
import pytest
import torch

import ftb
from tests.attn_cases import AttnCase, build, reference

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

