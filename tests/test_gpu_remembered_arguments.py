"""Options given as tensors: a call takes their value of the moment. The argument blocks that calls
remember are kept by value, so changing such a tensor in place must not bring the old one back."""
import pytest
import torch

import ftb
from tests.attn_cases import AttnCase, build
from tests.test_gpu_attention import attend

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


@pytest.mark.parametrize("device", ["cpu", "cuda"])
def test_norm_options(device):
    x, y = (torch.randn(5, 256, device="cuda").to(BF) for _ in range(2))
    w = torch.ones(256, dtype=BF, device="cuda")
    scale, eps = torch.tensor(0.5, device=device), torch.tensor(1e-6, device=device)
    for s, e in ((0.5, 1e-6), (2.0, 1e-6), (2.0, 0.5)):
        scale.fill_(s), eps.fill_(e)
        for a, b in zip(ftb.block_norm(x, y, scale=scale, pre_weight=w, eps=eps),
                        ftb.block_norm(x, y, scale=scale.item(), pre_weight=w, eps=eps.item())):
            assert torch.equal(a, b)
        assert torch.equal(ftb.rms_norm(x, w, eps), ftb.rms_norm(x, w, eps.item()))


@pytest.mark.parametrize("device", ["cpu", "cuda"])
def test_attention_options(device):
    c = AttnCase([(40, 300), (9, 9)])
    build(c)
    max_q, window = (torch.tensor(v, device=device) for v in (9, 50))
    scale, causal = torch.tensor(0.1, device=device), torch.tensor(True, device=device)
    for m, w, s, k in ((9, 50, 0.1, True), (40, 50, 0.1, True), (40, 7, 0.1, True),
                       (40, 7, 0.5, True), (40, 7, 0.5, False)):
        max_q.fill_(m), window.fill_(w), scale.fill_(s), causal.fill_(k)
        outs = [torch.full_like(c.t["q"], 3.0) for _ in range(2)]
        attend(c, max_q=max_q, window=window, scale=scale, causal=causal, out=outs[0])
        attend(c, max_q=m, window=w, scale=scale.item(), causal=k, out=outs[1])
        assert torch.equal(*outs), (m, w, s, k)
    with pytest.raises(ValueError, match="status 2"):  # max_q was 9 for 40 tokens; and cleared
        attend(c, max_q=40, check_status=True)


def test_sections():
    q = torch.randn(6, 4, 64, device="cuda").to(BF)
    at = torch.randint(0, 50, (3, 6), dtype=torch.int32, device="cuda")
    table = ftb.rope_table(50, 64)
    counts = torch.tensor([12, 10, 10])
    parts = tuple(counts)  # (its elements are views)
    for first in (12, 20):
        counts[0], counts[1] = first, 22 - first
        want = ftb.rope(q, q, at, table, sections=tuple(counts.tolist()))
        for sections in (counts, parts, counts.tolist()):
            for a, b in zip(ftb.rope(q, q, at, table, sections=sections), want):
                assert torch.equal(a, b)
