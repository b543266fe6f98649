"""ftb.DecoderLayer: its stages, and prompts in chunks and tokens against prompts at once.

Between two ways through the same layer each stage rounds to bf16 again: qkv, turned q and k, P and
the attention's output, o, r, h, the MoE layer's four and its output's residual. Each differs by at
most 2^-8 relative per element in norm from its exact value either way, so after 12 such stages by
at most 2 * 12 * 2^-8 of the norm even if every rounding pointed the same way; they do not, and the
square root of the count is the rule: 2 * sqrt(12) * 2^-8 < 2^-5.
"""
import os
import subprocess
import sys

import pytest
import torch

import ftb
from ftb import synth
from tests.conftest import ROOT

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def build(sections=None, window=0, seed=0, hidden=512, q_heads=8, kv_heads=2, D=64):
    g = torch.Generator().manual_seed(seed)

    def w(*shape, s=1.0, m=0.0):
        return (torch.randn(*shape, generator=g) * s + m).to(BF).cuda()

    bank = synth.make_bank(16, hidden, 256, seed=seed).to("cuda")
    # the router's choice hangs on the bias alone: a rounding must not change the experts
    moe = ftb.Nvfp4MoELayer(ftb.B200Nvfp4Experts(bank), 4, router="sigmoid",
                            gate_weight=(torch.randn(16, hidden, generator=g) * 0.01).cuda(),
                            score_bias=torch.arange(16.0).cuda() * 10)
    return ftb.DecoderLayer(
        w((q_heads + 2 * kv_heads) * D, hidden, s=hidden ** -0.5),
        w(hidden, q_heads * D, s=(q_heads * D) ** -0.5), moe, w(hidden, s=0.1, m=1.0),
        w(hidden, s=0.1, m=1.0), q_heads, kv_heads, ftb.rope_table(600, D),
        post_attn_norm=w(hidden, s=0.1, m=1.0), attn_gate=w(hidden, s=0.1, m=1.0),
        residual_scale=0.5, sections=sections, window=window)


def through(layer, cache, x, chunks, page, pages):
    """The layer over one sequence in chunks; (residual, hidden) of all tokens."""
    past, out = 0, []
    for n in chunks:
        step = ftb.AttnStep.build([pages], [past], [n], page)
        out.append(layer(x[past:past + n], None, step, cache, layer.input_norm))
        past += n
    return [torch.cat(t) for t in zip(*out)]


@pytest.mark.parametrize("window", [0, 100])
@pytest.mark.parametrize("chunks", [[180, 1, 1, 1], [1] * 20, [64, 65, 7]])
def test_chunks_agree_with_the_prompt_at_once(chunks, window):
    layer = build(window=window)
    total = sum(chunks)
    x = torch.randn(total, 512, generator=torch.Generator().manual_seed(5)).to(BF).cuda()
    pages = [5, 0, 3, 9, 1, 7, 2, 8, 4, 6, 10, 11, 12]
    whole = through(layer, ftb.PagedKvCache(13, 16, 2, 64), x, [total], 16, pages)
    parts = through(layer, ftb.PagedKvCache(13, 16, 2, 64), x, chunks, 16, pages)
    for a, b in zip(whole, parts):
        assert torch.isfinite(a).all()
        d = (a.float() - b.float()).norm() / a.float().norm()
        assert d <= 2.0 ** -5, d


def test_layer_is_its_operators():
    """The layer's result is that of the public calls in its order."""
    layer = build(sections=(12, 10, 10))
    prompts = [70, 5, 33]
    pages = [[0, 1, 2], [3], [4, 5]]
    positions = torch.randint(0, 600, (3, sum(prompts)), dtype=torch.int32, device="cuda")
    step = ftb.AttnStep.build(pages, [0, 0, 0], prompts, 32, positions=positions)
    x = torch.randn(sum(prompts), 512, device="cuda").to(BF)
    cache = ftb.PagedKvCache(6, 32, 2, 64)
    r, h = layer(x, None, step, cache, layer.input_norm)
    n = ftb.rms_norm(x, layer.input_norm)
    q, k, v = (n @ layer.qkv.t()).view(-1, 12, 64).split([8, 2, 2], 1)
    again = ftb.PagedKvCache(6, 32, 2, 64)
    q = ftb.rope_append(q, k, v, positions, layer.rope_table, again.k, again.v, step.slots,
                        sections=(12, 10, 10))
    assert torch.equal(again.k, cache.k) and torch.equal(again.v, cache.v)
    a = ftb.paged_attention(q, cache.k, cache.v, step.block_table, step.kv_len, step.cu_q, 70)
    r2, h2 = ftb.block_norm(x, a.view(-1, 512) @ layer.o.t(), post_weight=layer.post_attn_norm,
                            gate=layer.attn_gate, scale=0.5, pre_weight=layer.moe_norm)
    r2, h2 = ftb.block_norm(r2, layer.moe(h2), scale=0.5, pre_weight=layer.input_norm)
    assert torch.equal(r, r2) and torch.equal(h, h2)


def test_residual_in_32_bits():
    layer = build()
    step = ftb.AttnStep.build([[0, 1]], [0], [40], 32)
    x = torch.randn(40, 512, device="cuda")
    r, h = layer(x, None, step, ftb.PagedKvCache(2, 32, 2, 64), layer.input_norm)
    assert r.dtype == torch.float32 and h.dtype == BF and torch.isfinite(r).all()


def test_example_runs():
    out = subprocess.run([sys.executable, os.path.join(ROOT, "examples", "decoder_layers.py"),
                          "--tokens", "200", "--steps", "3"], capture_output=True, text=True,
                         timeout=300)
    assert out.returncode == 0, out.stderr
    assert "step 3: 4 new tokens over" in out.stdout
