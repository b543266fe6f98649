"""Two decoder layers with random weights: packed prompts of different lengths, then decode steps.

    python examples/decoder_layers.py [--tokens 600] [--steps 16]

Each layer runs norm, qkv projection, rotary positions with the cache write, paged attention,
output projection, gated residual and norm, and the NVFP4 MoE layer (2048 hidden, 768 expert
intermediate, 64 experts, top-8). Prints the time per step.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "..",
                                "freetoken-ox-boost_b200"))
import ftb  # noqa: E402
from ftb import synth  # noqa: E402


def build_layer(seed: int, hidden=2048, inter=768, experts=64, top_k=8, q_heads=16, kv_heads=4,
                head_dim=128, positions=1024):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def weight(*shape, scale):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).bfloat16()

    def ones():
        return torch.ones(hidden, dtype=torch.bfloat16, device="cuda")

    bank = synth.make_bank(experts, hidden, inter, seed=seed).to("cuda")
    moe = ftb.Nvfp4MoELayer(ftb.B200Nvfp4Experts(bank), top_k,
                            gate_weight=weight(experts, hidden, scale=hidden ** -0.5).float())
    return ftb.DecoderLayer(
        weight((q_heads + 2 * kv_heads) * head_dim, hidden, scale=hidden ** -0.5),
        weight(hidden, q_heads * head_dim, scale=(q_heads * head_dim) ** -0.5), moe, ones(), ones(),
        q_heads, kv_heads, ftb.rope_table(positions, head_dim), post_attn_norm=ones(),
        post_moe_norm=ones(), residual_scale=0.5)


def run(layers, caches, residual, step):
    hidden = None
    for i, (layer, cache) in enumerate(zip(layers, caches)):
        following = layers[i + 1].input_norm if i + 1 < len(layers) else layers[0].input_norm
        residual, hidden = layer(residual, hidden, step, cache, following)
    return hidden


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--tokens", type=int, default=600, help="length of the longest prompt")
    ap.add_argument("--steps", type=int, default=16, help="decode steps after the prompts")
    args = ap.parse_args()
    page = 64
    layers = [build_layer(i, positions=args.tokens + args.steps) for i in range(2)]
    prompts = [args.tokens, max(1, args.tokens // 3), max(1, args.tokens // 7), 1]
    need = [-(-(n + args.steps) // page) for n in prompts]
    ids = torch.randperm(sum(need)).tolist()
    pages = [[ids.pop() for _ in range(n)] for n in need]
    caches = [ftb.PagedKvCache(sum(need), page, 4, 128) for _ in layers]
    past, new = [0] * len(prompts), prompts
    start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    for i in range(1 + args.steps):
        step = ftb.AttnStep.build(pages, past, new, page)
        x = torch.randn(sum(new), 2048, device="cuda").bfloat16()
        start.record()
        hidden = run(layers, caches, x, step)
        end.record()
        torch.cuda.synchronize()
        assert torch.isfinite(hidden).all()
        if i in (0, args.steps):
            print(f"step {i}: {sum(new)} new tokens over {sum(past)} cached ones, "
                  f"{start.elapsed_time(end):.3f} ms")
        past, new = [p + n for p, n in zip(past, new)], [1] * len(prompts)


if __name__ == "__main__":
    main()
