"""The q that ftb.rope_append returns beside an 8-bit cache, element by element: products and sums are single
operations in 32 bits there as in tests/fp8_cases.py, rounded once to q's type, so the numbers are equal."""
import math

import pytest
import torch

from tests.fp8_cases import turned
from tests.test_gpu_fp8_append import call, make

BF, F16 = torch.bfloat16, torch.float16


def assert_same(got, want):
    """NaN in the same places, equal numbers in all others."""
    assert got.dtype == want.dtype and got.shape == want.shape
    nan = want.isnan()
    assert torch.equal(got.isnan(), nan)
    assert torch.equal(got[~nan], want[~nan])


def turned_q(c):
    q = c["qkv"][:, :c["heads"][0]]
    return turned(q, c["positions"], c["table"], c["pairs"], c["sections"], c["order"]).to(q.dtype)


def check_q(c):
    want = turned_q(c)
    assert want[~want.isnan()].ne(0).any() or not want.numel()
    assert_same(call(c)["q"], want)


@pytest.mark.parametrize("dtype", [BF, F16])
def test_one_wrong_number_is_seen(dtype):
    """(on the CPU: the other tests' comparison against an oracle with a mistake in it)"""
    c = make(9, range(9), dtype=dtype)
    c["positions"][3] = -1
    want = turned_q(c)
    assert want[3].isnan().all() and not want[:3].isnan().any()
    assert_same(want.clone(), want)
    for at, to in (((0, 0, 0), 1.5), ((8, 3, 63), math.inf), ((4, 1, 5), math.nan), ((3, 2, 7), 0.0)):
        bad = want.clone()
        bad[at] = to
        with pytest.raises(AssertionError):
            assert_same(bad, want)
    for bad in (dict(c, pairs="adjacent"), dict(c, positions=c["positions"].roll(1))):
        with pytest.raises(AssertionError):
            assert_same(turned_q(bad), want)


# vectors of 8, 4 and 1 elements; heads of which all, or a part, is turned
SHAPES = [(128, 128, "half"), (128, 64, "adjacent"), (80, 48, "adjacent"), (112, 112, "half"),
          (64, 24, "half"), (72, 20, "half"), (72, 40, "half"), (66, 6, "adjacent"), (16, 16, "half"),
          (256, 128, "half"), (512, 256, "adjacent")]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("D,rot,pairs", SHAPES)
@pytest.mark.parametrize("tokens", [1, 40, 600, 1100, 2100, 4099])
def test_heads_and_rotations(D, rot, pairs, tokens, dtype):
    check_q(make(tokens, range(7, 7 + tokens), D=D, rot=rot, pairs=pairs, pages=140, dtype=dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("heads", [(1, 1), (3, 1), (8, 8), (40, 5), (33, 1), (130, 2)])
@pytest.mark.parametrize("tokens", [1, 5, 64, 4095, 4096, 4097, 4103, 5000])
def test_head_counts_and_tokens(heads, tokens):
    """(from 4096 tokens on, eight tokens to a thread block)"""
    check_q(make(tokens, range(3, 3 + tokens), heads=heads, pages=160, D=32, rot=32, seed=tokens))


@pytest.mark.gpu
@pytest.mark.parametrize("pairs", ["half", "adjacent"])
@pytest.mark.parametrize("axes,sections,order", [(3, (12, 10, 10), "cyclic"), (2, (32, 0), "blocks"),
                                                 (4, (8, 8, 8, 8), "blocks"), (3, (5, 20, 7), "blocks"),
                                                 (4, (14, 6, 6, 6), "cyclic")])
def test_axes(axes, sections, order, pairs):
    for tokens in (9, 530, 2100, 4101):
        check_q(make(tokens, range(20, 20 + tokens), axes=axes, sections=sections, order=order, pages=140,
                     pairs=pairs))


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [20, 4100])
def test_numbers_and_positions_at_the_limits(tokens):
    for dtype, big in ((BF, 2.0 ** 120), (F16, 30000.0)):
        c = make(tokens, range(tokens), dtype=dtype, pages=140)
        x = c["qkv"]
        x[2] *= big
        x[5, 1, 3], x[6, 0, 40], x[7, 3, 0] = math.inf, -math.inf, math.nan
        x[8] = 2.0 ** -24 if dtype == F16 else 2.0 ** -130
        c["positions"][3], c["positions"][4] = 500, -1
        check_q(c)
