"""ftb.paged_attention over an 8-bit cache: scales of blocks that no token sees (new pages have 0) leave the
outputs as they are, bit for bit."""
import pytest
import torch

import ftb
from tests.fp8_cases import Fp8Case, build

pytestmark = pytest.mark.gpu
BF, F16 = torch.bfloat16, torch.float16


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("head", [64, 128])
@pytest.mark.parametrize("pairs,window,page", [
    ([(1, 70), (1, 3), (1, 300)], 0, 64), ([(1, 5000)] * 3, 1000, 64), ([(4, 70), (3, 33)], 0, 64),
    ([(40, 40), (17, 17), (90, 90)] * 20, 0, 128), ([(40, 70)] * 60, 0, 256), ([(300, 1001)] * 8, 0, 64),
    ([(900, 2000), (300, 700), (3, 3)], 100, 64), ([(700, 1500)] * 3, 333, 128)])
def test_blocks_that_no_token_sees(pairs, window, page, head, dtype):
    c = Fp8Case(pairs, q_heads=16, page=page, block=16, head=head, window=window, dtype=dtype)
    build(c)  # scales of NaN behind a sequence's keys, of infinity below every token's window

    def outputs(low):
        t = {n: torch.where(x.isfinite(), x, low) if "scale" in n else x for n, x in c.t.items()}
        return ftb.paged_attention(**t, window=window, return_lse=True, check_status=True)

    out, lse = outputs(2.0 ** -7)
    for low in (0.0, 2.0 ** -40, 2.0 ** 40, float("nan")):
        got = outputs(low)
        assert torch.equal(out, got[0]) and torch.equal(lse, got[1])
