"""What the streaming kernel of ftb.paged_attention keeps beyond the bounds of tests/attn_cases.py:
its weights are two operands, the weight in the tensors' type and the rest of that rounding, so an
output's error is its own rounding.

Bounds, with u the unit roundoff of the type, A = sum p_j |v_j| over the softmax p, N keys:
  u |o|        the output's rounding
  u^2 A        the rounding of the rest
  2^-13 A      scores and exponentials, as in tests/attn_cases.py (2^-14 A for all of fp32's part where
               scores are exact: an exponential to 2^-21, at most 2^9 steps of 2^-23 in each sum)
  f16 only:    a weight's own subnormals, 2^-25 of the largest each: 2^-25 sum |v_j| / l, and the
               output's, 2^-25."""
import math

import pytest
import torch

import ftb
from tests.attn_cases import U, AttnCase, build

pytestmark = pytest.mark.gpu
BF, F16 = torch.bfloat16, torch.float16


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("kv", [2, 100, 1024, 20000])
@pytest.mark.parametrize("n", [1, 4])
def test_weights_that_all_round_the_same_way(kv, dtype, n):
    """Half of the keys have weight 1 and V 1, the others a weight as far between two numbers of the
    type as scores allow, and V so that the sum nearly vanishes: rounded once, the weights would
    be off by many times the bound."""
    s = -torch.arange(0.5, 0.7, 2.0 ** -13, dtype=torch.float64)
    s = s[s.to(dtype).double() == s]  # scores of the type
    off = (s.exp().to(dtype).double() / s.exp() - 1).abs()
    score = s[off.argmax()].item()
    p = math.exp(score)
    v = torch.tensor(-1 / p, dtype=torch.float64).to(dtype).item()
    c = AttnCase([(n, kv)], dtype=dtype, causal=False, scale=1.0, page=64)
    build(c)
    c.t["q"].zero_()
    c.t["q"][..., 0] = 1.0
    table = c.t["block_table"][0, :-(-kv // 64)].long()
    key = torch.zeros(64, 1, 128, dtype=dtype, device="cuda")
    key[1::2, :, 0] = score
    c.t["k_cache"][table] = key
    value = torch.ones(64, 1, 1, dtype=dtype, device="cuda")
    value[1::2] = v
    c.t["v_cache"][table] = value
    ones, others = (kv + 1) // 2, kv // 2
    l = ones + others * p
    want, total = (ones + others * p * v) / l, (ones - others * p * v) / l
    u = U[dtype]
    bound = u * abs(want) + (u * u + 2.0 ** -14) * total + 2.0 ** -25
    if dtype == F16:
        bound += 2.0 ** -25 * (ones - others * v) / l
    once = torch.tensor(p, dtype=torch.float64).to(dtype).item()
    assert abs((ones + others * once * v) / l - want) > 2 * bound
    out = ftb.paged_attention(**c.t, causal=False, scale=1.0)
    assert (out.double() - want).abs().max().item() <= bound


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("pairs,head,window", [([(1, 1)], 128, 0), ([(1, 129), (1, 64)], 80, 0),
                                               ([(1, 1000)], 128, 300), ([(4, 9), (3, 700)], 64, 0),
                                               ([(1, 9000), (1, 15000)], 128, 0),
                                               ([(2, 3000)], 64, 2000)])
def test_random_inputs(pairs, head, window, dtype):
    c = AttnCase(pairs, head=head, window=window, dtype=dtype, page=32, seed=7)
    q, keys = build(c)
    out = ftb.paged_attention(**c.t, window=window).double().cpu()
    u, at = U[dtype], 0
    for (n, kv), x in zip(c.pairs, keys):
        place, j = torch.arange(kv - n, kv)[:, None], torch.arange(kv)
        seen = (j <= place) & ((j > place - window) if window else True)
        for h in range(c.q_heads):
            k, v = (x[:, i, h // 4].double() for i in range(2))
            s = (q[at:at + n, h].double() @ k.t() * head ** -0.5).masked_fill(~seen, -math.inf)
            p = (s - s.amax(1, keepdim=True)).exp()
            l = p.sum(1, keepdim=True)
            want, total = p @ v / l, p @ v.abs() / l
            bound = u * want.abs() + (u * u + 2.0 ** -13) * total + 1e-30
            if dtype == F16:
                bound += 2.0 ** -25 * (seen.double() @ v.abs()) / l + 2.0 ** -25
            worst = ((out[at:at + n, h] - want).abs() / bound).max().item()
            assert worst <= 1.0, worst
        at += n
