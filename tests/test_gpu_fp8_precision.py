"""What the few-row kernels of ftb.paged_attention keep of an 8-bit cache beyond the bounds of
tests/fp8_cases.py: their weights are two operands in every type of q, the weight in f16 and the rest of that
rounding.

Bound, with u the unit roundoff of q's type and A = sum p_j |v_j| over the softmax p:
  u |o|     the output's rounding
  2^-22 A   the rounding of the rest
  2^-14 A   fp32's part where scores are exact: an exponential to 2^-21, at most 2^9 steps of 2^-23 in
            each sum
  2^-25     f16 only: the output's subnormals"""
import math

import pytest
import torch

import ftb
from tests.attn_cases import U
from tests.fp8_cases import FP8, Fp8Case, build

pytestmark = pytest.mark.gpu
BF, F16 = torch.bfloat16, torch.float16


def worst_weight(dtype):
    """(score, code of V): a score of the type whose weight p lies as far between two numbers of f16 as any
    whose p v all but cancels 1."""
    best = (0.0,)
    for v in (-1.125, -1.25, -1.375, -1.5, -1.625, -1.75, -1.875):
        s = torch.arange(-8, 9, dtype=torch.float64) * 2.0 ** -11 - math.log(-v)
        s = s.to(dtype).double()
        p = s.exp()
        s = s[(1 + p * v).abs() < 2.0 ** -9]
        off = (s.exp().half().double() - s.exp()).abs() * -v / (1 + s.exp())
        if off.numel() and off.max() > best[0]:
            best = (off.max().item(), s[off.argmax()].item(), v)
    return best[1:]


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("kv", [2, 100, 1024, 20000])
@pytest.mark.parametrize("n,batch", [(1, 1), (1, 90), (2, 1), (4, 1), (4, 3)])
def test_weights_that_all_round_the_same_way(kv, dtype, n, batch):
    """Half of the keys have weight 1 and V 1, the others one that f16 misses by half a step, and V so that
    the sum nearly vanishes: a weight rounded once would be off by more than twice the bound. (4, 8 and 16
    rows per kv head, one head at a time and pairs of them.)"""
    if batch == 90 and kv == 20000:
        kv = 3000
    score, v = worst_weight(dtype)
    p = math.exp(score)
    c = Fp8Case([(n, kv)] * batch, dtype=dtype, causal=False, scale=1.0, page=64, block=64)
    build(c)
    c.t["q"].zero_()
    c.t["q"][..., 0] = score
    key = torch.zeros(64, 1, 128, device="cuda")
    key[1::2, :, 0] = 1.0
    value = torch.ones(64, 1, 1, device="cuda")
    value[1::2] = v
    for name, x in (("k", key), ("v", value)):
        c.t[name + "_cache"].copy_(x.to(FP8).expand_as(c.t[name + "_cache"][0]))
        c.t[name + "_scale"].fill_(1.0)
    ones, others = (kv + 1) // 2, kv // 2
    l = ones + others * p
    want, total = (ones + others * p * v) / l, (ones - others * p * v) / l
    bound = U[dtype] * abs(want) + (2.0 ** -22 + 2.0 ** -14) * total + (2.0 ** -25 if dtype == F16 else 0)
    once = torch.tensor(p, dtype=torch.float64).half().double().item()
    assert abs((ones + others * once * v) / l - want) > 2 * bound
    out = ftb.paged_attention(**c.t, causal=False, scale=1.0)
    assert (out.double() - want).abs().max().item() <= bound
