"""ftb.paged_attention at the ends of its arguments' ranges."""
import pytest
import torch

import ftb
from tests.attn_cases import AttnCase, build
from tests.test_gpu_attention import attend

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("pairs", [[(5, 70), (3, 3)], [(400, 900), (129, 129)]])
def test_bounds_past_32_bits(pairs):
    c = AttnCase(pairs)
    build(c)
    want = attend(c)
    for max_q in (2 ** 31 - 1, 2 ** 31, 2 ** 32, 2 ** 40):
        out = torch.full_like(want, 3.0)
        attend(c, max_q=max_q, out=out)
        assert torch.equal(out, want), max_q
    for window in (2 ** 31 - 1, 2 ** 31, 2 ** 32 + 1, 2 ** 63):
        assert torch.equal(attend(c, window=window), want), window
    with pytest.raises(ValueError, match="max_q"):
        attend(c, max_q=-1)


@pytest.mark.parametrize("pairs", [[(9, 4), (3, 70)], [(300, 200), (40, 1000)]])
def test_a_window_that_reaches_every_key_is_no_window(pairs):
    """Tokens before the first key too, which see every key where the mask is not causal."""
    for causal in (True, False):
        c = AttnCase(pairs, causal=causal)
        build(c)
        want = attend(c, causal=causal)
        for window in (1300, 2 ** 31 - 1):
            assert torch.equal(attend(c, causal=causal, window=window), want)


def test_more_row_tiles_than_a_grid_holds():
    """128 heads over one, 8200 tokens by max_q (a loose bound): 65600 tiles of 16 rows of little
    work each."""
    c = AttnCase([(8, 8)] * 1025, q_heads=128, kv_heads=1, head=8, page=8)
    build(c)
    want = attend(c)
    got = attend(c, max_q=8200)
    # each way is within an output's and the weights' rounding of the definition: 2 * 2 * 2^-8 of
    # values that reach 4, and a little for the scores
    assert (got.float() - want.float()).abs().max() <= 2.0 ** -3
    # a window of one key: each token gets its own V row (the first 7 see none), whose weight is
    # rounded against a sum that is not: 2^-8 of it, and as much for the output
    c = AttnCase([(8200, 8193)], q_heads=128, kv_heads=1, head=8, page=8)
    _, keys = build(c)
    out = attend(c, window=1).cpu()
    v = keys[0][:, 1].float()
    assert (out[:7] == 0).all()
    assert ((out[7:].float() - v).abs() <= 2.0 ** -7 * 1.01 * v.abs()).all()


def test_a_batch_beyond_the_plan():
    """25700 sequences of 2 tokens of 16 heads over one: with half of them each, the other kernel."""
    batch = 25700
    c = AttnCase([(2, 9)] * batch, q_heads=32, kv_heads=2, head=64, page=8)
    build(c)
    got = attend(c)
    half = batch // 2
    for part in (slice(0, half), slice(half, batch)):
        rows = slice(2 * part.start, 2 * part.stop)
        cu = c.t["cu_q"][part.start:part.stop + 1] - 2 * part.start
        want = attend(c, q=c.t["q"][rows], block_table=c.t["block_table"][part],
                      kv_len=c.t["kv_len"][part], cu_q=cu)
        # each within an output's and the weights' rounding of the definition, of values up to 5
        assert (got[rows].float() - want.float()).abs().max() <= 4 * 5 * 2.0 ** -8


def test_table_without_a_column():
    """No sequence has a key: outputs 0, lse -inf."""
    for n in (1, 40):
        q = torch.randn(2 * n, 8, 64, device="cuda").bfloat16()
        cache = torch.zeros(3, 16, 2, 64, dtype=torch.bfloat16, device="cuda")
        table = torch.zeros(2, 0, dtype=torch.int32, device="cuda")
        lens = torch.zeros(2, dtype=torch.int32, device="cuda")
        cu = None if n == 1 else torch.tensor([0, n, 2 * n], dtype=torch.int32, device="cuda")
        out, lse = ftb.paged_attention(q, cache, cache, table, lens, cu, n, return_lse=True,
                                       check_status=True)
        assert (out == 0).all() and torch.isneginf(lse).all()
