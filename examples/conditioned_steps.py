"""Denoising steps conditioned by cross attention, the prompts' keys and values held in 8 bits.

A guided batch (a prompt and the empty prompt) attends to its text states at every step.  The states are projected once
and written into an 8-bit cache; each step reads the cache.  Then one training step of the attention with dense keys and
values, and a few of the whole layer (layer norm, rotary positions, Muon for its matrices), which is quantised at the end.

    python examples/conditioned_steps.py [--tokens 4096] [--steps 4]
"""
from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

from minixmax_h3_b200 import ops  # noqa: E402
from minixmax_h3_b200.attention import cross_attention  # noqa: E402
from minixmax_h3_b200.block import CrossAttention, RopeSpec, TrainableCrossAttention, load_quant_linear  # noqa: E402
from minixmax_h3_b200.optim import Muon  # noqa: E402


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__)
    ap.add_argument("--tokens", type=int, default=4096, help="video tokens of a sample")
    ap.add_argument("--text", type=int, default=300, help="text tokens of the prompt")
    ap.add_argument("--steps", type=int, default=4)
    a = ap.parse_args()
    dev, hidden, heads, cond_dim = "cuda", 1024, 8, 4096
    gen = torch.Generator(device=dev).manual_seed(0)
    layer = CrossAttention(hidden, heads, 128, cond_dim, kv_heads=4, device=dev)
    for ql in (layer.q_proj, layer.kv_proj, layer.out_proj):
        w = torch.randn(ql.out_features, ql.in_features, generator=gen, device=dev) * 0.02
        load_quant_linear(ql, w, "int8_tensorwise")

    text = torch.randn(2, a.text, cond_dim, generator=gen, device=dev).to(torch.bfloat16)
    text_lens = torch.tensor([a.text, 0], dtype=torch.int32, device=dev)  # the second sample has no prompt
    blocks = (a.text + 63) // 64
    cache = ops.KV8Cache.empty(2 * blocks, layer.kv_heads, 128, device=dev)
    table = torch.arange(2 * blocks, dtype=torch.int32, device=dev).view(2, blocks)
    layer.fill(cache, text, table, torch.zeros_like(text_lens), new_lens=text_lens)

    x = torch.randn(2, a.tokens, hidden, generator=gen, device=dev).to(torch.bfloat16)
    for step in range(a.steps):
        x = x + layer(x, cache=cache, block_table=table, cond_lens=text_lens)
    dense = layer(x, text, cond_lens=text_lens)
    cached = layer(x, cache=cache, block_table=table, cond_lens=text_lens)
    off = ((cached - dense).float().norm() / dense.float().norm()).item()
    print(f"{a.steps} steps of 2 x {a.tokens} tokens over {a.text} + 0 text tokens; 8-bit against 16-bit keys and values: "
          f"relative difference {off:.4f}")

    q = torch.randn(2, a.tokens, heads, 128, generator=gen, device=dev).to(torch.bfloat16).requires_grad_()
    k, v = (t.detach().requires_grad_() for t in layer.encode(text))
    loss = cross_attention(q, k, v, kv_lens=text_lens).float().square().mean()
    loss.backward()
    print(f"loss {loss.item():.5f}, |dq| {q.grad.float().norm().item():.3e}, |dk| {k.grad.float().norm().item():.3e}, "
          f"|dv| {v.grad.float().norm().item():.3e}")

    # video tokens by their places on a grid, text tokens along its first axis
    rope = ops.Rotary.build((44, 42, 42), device=dev)
    side = max(1, round((a.tokens / 4) ** 0.5))
    positions = RopeSpec.grid_positions(-(-a.tokens // (side * side)), side, side)[:a.tokens].to(dev, torch.int32)
    text_positions = torch.zeros(a.text, 3, dtype=torch.int32, device=dev)
    text_positions[:, 0] = torch.arange(a.text, device=dev)
    trained = TrainableCrossAttention(hidden, heads, 128, cond_dim, kv_heads=4, rope=rope, device=dev)
    matrices, rest = Muon(trained.matrices(), lr=0.01), torch.optim.AdamW(trained.norm.parameters(), lr=1e-3)
    target = torch.randn(2, a.tokens, hidden, generator=gen, device=dev)
    where = {"cond_lens": text_lens, "positions": positions, "cond_positions": text_positions}
    for step in range(a.steps):
        loss = (trained(x, text, **where).float() - target).square().mean()
        loss.backward()
        for opt in (matrices, rest):
            opt.step()
            opt.zero_grad()
        print(f"training step {step}: loss {loss.item():.5f}")
    with torch.no_grad():
        dense = trained(x, text, **where)
        off = ((trained.quantized()(x, text, **where) - dense).float().norm() / dense.float().norm()).item()
    print(f"the trained layer in 8 bits against 16: relative difference {off:.4f}")


if __name__ == "__main__":
    main()
