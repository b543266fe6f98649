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
