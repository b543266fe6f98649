"""The 8-bit cache's operators together: a decoder layer over it against their calls one by one and
against a 16-bit cache, and sequences that are forked, extended, compacted and freed between steps.

Against the 16-bit cache: an element of K or V held in e4m3 is off by at most 2^-4 of itself (half a step
of 2^-3), uniformly over about its range, so by 2^-4 / sqrt(3) in norm. The attention's output is a sum of
V's errors with the weights of a softmax over scores whose own errors are 2^-4 / sqrt(3) sqrt(2) |q||k|
scale / sqrt(D) in norm: with normalised q and k of size 1 the weights move by 2^-4 relative, no more than
V does. o is so within 2^-3 of the attention's norm, and the residual stream, which has the attention's
part with a factor of 1/2 beside itself, within 2^-4; the norm and the MoE layer may double it."""
import os
import subprocess
import sys

import pytest
import torch

import ftb
from tests.conftest import ROOT
from tests.test_gpu_decoder import build

pytestmark = pytest.mark.gpu
BF, F8 = torch.bfloat16, torch.float8_e4m3fn


def test_layer_is_its_operators():
    layer = build()
    prompts, pages = [70, 5, 33], [[0, 1, 2], [3], [4, 5]]
    step = ftb.AttnStep.build(pages, [0, 0, 0], prompts, 32)
    x = torch.randn(sum(prompts), 512, device="cuda").to(BF)
    cache, again = (ftb.PagedKvCache(6, 32, 2, 64, dtype=F8, scale_block=16) for _ in range(2))
    r, h = layer(x, None, step, cache, layer.input_norm)
    n = ftb.rms_norm(x, layer.input_norm)
    q, k, v = (n @ layer.qkv.t()).view(-1, 12, 64).split([8, 2, 2], 1)
    scales = dict(k_scale=again.k_scale, v_scale=again.v_scale)
    q = ftb.rope_append(q, k, v, step.positions, layer.rope_table, again.k, again.v, step.slots, **scales)
    for a, b in zip(cache.tensors(), again.tensors()):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    a = ftb.paged_attention(q, again.k, again.v, step.block_table, step.kv_len, step.cu_q, 70, **scales)
    r2, h2 = ftb.block_norm(x, a.view(-1, 512) @ layer.o.t(), post_weight=layer.post_attn_norm,
                            gate=layer.attn_gate, scale=0.5, pre_weight=layer.moe_norm)
    r2, h2 = ftb.block_norm(r2, layer.moe(h2), scale=0.5, pre_weight=layer.input_norm)
    assert torch.equal(r, r2) and torch.equal(h, h2)


@pytest.mark.parametrize("chunks", [[183], [60, 100, 1, 1, 1]])
def test_close_to_a_16_bit_cache(chunks):
    layer = build(seed=2)
    x = torch.randn(sum(chunks), 512, generator=torch.Generator().manual_seed(5)).to(BF).cuda()
    out = []
    for kw in (dict(), dict(dtype=F8)):
        cache, past, parts = ftb.PagedKvCache(6, 32, 2, 64, **kw), 0, []
        for n in chunks:
            step = ftb.AttnStep.build([[5, 0, 3, 1, 2, 4]], [past], [n], 32)
            parts.append(layer(x[past:past + n], None, step, cache)[0])
            past += n
        out.append(torch.cat(parts).float())
    assert (out[0] - out[1]).norm() / out[0].norm() <= 2.0 ** -3
    assert not torch.equal(*out)


def test_forked_and_compacted_sequences_decode_as_if_alone():
    """Two continuations of one prompt, and another sequence, through a pool: each as it would be in a
    cache of its own, since its tokens join the same blocks in the same order there."""
    layer, page = build(seed=3), 32
    g = torch.Generator().manual_seed(8)
    prompts = [torch.randn(n, 512, generator=g).to(BF).cuda() for n in (75, 40)]
    tails = [torch.randn(n, 512, generator=g).to(BF).cuda() for n in (30, 30, 30)]
    cache = ftb.PagedKvCache(24, page, 2, 64, dtype=F8)
    pool = ftb.PagePool(24, page, [cache])
    junk = pool.allocate(5)  # so that there is something to compact
    a, b = [], []
    pool.extend([a, b], [0, 0], [75, 40])
    layer(torch.cat(prompts), None, ftb.AttnStep.build([a, b], [0, 0], [75, 40], page), cache)
    c = pool.fork(a)
    pool.free(junk)
    seqs, past, got = [a, c, b], [75, 75, 40], [[], [], []]
    for i in range(30):
        pool.extend(seqs, past, [1, 1, 1])
        if i == 12:
            assert pool.compact(seqs) > 0
        step = ftb.AttnStep.build(seqs, past, [1, 1, 1], page)
        y, _ = layer(torch.stack([t[i] for t in tails]), None, step, cache)
        for s, row in zip(got, y):
            s.append(row)
        past = [p + 1 for p in past]
    assert not set(a[2:]) & set(c[2:]) and a[:2] == c[:2]
    # each on its own, beside two others, so that the steps have the same shapes
    alone = ftb.PagedKvCache(24, page, 2, 64, dtype=F8)
    pages = [list(range(i * 4, i * 4 + 4)) for i in range(3)]
    for ids, p in zip(pages, (0, 0, 1)):
        n = len(prompts[p])
        layer(prompts[p], None, ftb.AttnStep.build([ids], [0], [n], page), alone)
    past = [75, 75, 40]
    for i in range(30):
        step = ftb.AttnStep.build(pages, past, [1, 1, 1], page)
        y, _ = layer(torch.stack([t[i] for t in tails]), None, step, alone)
        for s, row in zip(got, y):
            # (the prompts' projections have other shapes: their roundings may differ)
            assert (s[i].float() - row.float()).norm() / row.float().norm() <= 2.0 ** -4
        past = [p + 1 for p in past]
    for ids in seqs:
        pool.free(ids)
    assert pool.free_pages == 24


def test_example_runs():
    out = subprocess.run([sys.executable, os.path.join(ROOT, "examples", "decoder_layers.py"), "--tokens",
                          "200", "--steps", "3", "--cache", "e4m3", "--samples", "2"],
                         capture_output=True, text=True, timeout=300)
    assert out.returncode == 0, out.stderr
    assert "step 3: 8 new tokens over" in out.stdout
