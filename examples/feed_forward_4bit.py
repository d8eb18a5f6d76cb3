"""Train with the fused gated feed-forward block, then serve in 4 bits.

A small random-init Qwen3 text tower takes a few optimizer steps that pull paired
sequences together, with every layer's feed-forward block as the fused kernels
of ``ops.ffn`` (forward and backward). The trained tower is then swapped to 4-bit
weights (``models.quantize_linears_fp4``: NVFP4 or MXFP4, activations quantised
on the way into every product) and embeds the same sequences; the script
prints the loss, how far the 4-bit embeddings turned, and the time of both.

    python examples/feed_forward_4bit.py [--fmt nvfp4|mxfp4] [--steps N]
"""

from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from representax_b200.models import quantize_linears_fp4
from representax_b200.models.qwen3 import Qwen3TextConfig, Qwen3TextTower, last_token_rows
from representax_b200.ops import nn as N


def embed(tower, ids, seg, pos):
    rows = tower(tower.token_embeddings(ids, torch.bfloat16), seg, pos)[last_token_rows(seg)]
    return torch.nn.functional.normalize(rows.float(), dim=-1)


def timed(fn, repeats: int = 20) -> float:
    """Milliseconds of one call on the device."""

    for _ in range(3):
        fn()
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    start.record()
    for _ in range(repeats):
        fn()
    end.record()
    torch.cuda.synchronize()
    return start.elapsed_time(end) / repeats


def main() -> None:
    parser = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    parser.add_argument("--fmt", choices=("nvfp4", "mxfp4"), default="nvfp4")
    parser.add_argument("--steps", type=int, default=8)
    args = parser.parse_args()
    device = torch.device("cuda", 0)
    gen = torch.Generator().manual_seed(0)
    cfg = Qwen3TextConfig(vocab_size=4096, hidden_size=512, intermediate_size=1408, num_hidden_layers=4,
                          num_attention_heads=8, num_key_value_heads=4, head_dimension=64)
    tower = Qwen3TextTower(cfg, gen).to(device).to(torch.bfloat16)
    # pairs of sequences that have nothing in common yet
    lengths = torch.randint(24, 200, (64,), generator=gen).tolist()
    rows = [torch.randint(0, cfg.vocab_size, (n,), generator=gen) for n in lengths]
    seg = N.Segments.from_lengths([len(r) for r in rows], device)
    ids = torch.cat(rows).to(device)
    pos = torch.cat([torch.arange(len(r)) for r in rows]).to(device)

    optimizer = torch.optim.AdamW(tower.parameters(), lr=1e-3)
    with N.fused_feed_forward():
        for step in range(args.steps):
            e = embed(tower, ids, seg, pos)
            loss = torch.nn.functional.cross_entropy(20 * e[:32] @ e[32:].T, torch.arange(32, device=device))
            optimizer.zero_grad()
            loss.backward()
            optimizer.step()
            print(f"step {step}: loss {loss.item():.4f}")
        with torch.no_grad():
            before = embed(tower, ids, seg, pos)
            bf16_ms = timed(lambda: embed(tower, ids, seg, pos))
    quantize_linears_fp4(tower, fmt=args.fmt)
    with torch.no_grad():
        after = embed(tower, ids, seg, pos)
        fp4_ms = timed(lambda: embed(tower, ids, seg, pos))
    cosine = (before * after).sum(-1)
    print(f"{args.fmt}: cosine to the bf16 embeddings mean {cosine.mean().item():.4f}, least {cosine.min().item():.4f}")
    print(f"embedding {seg.total} tokens: bf16 {bf16_ms:.3f} ms, {args.fmt} {fp4_ms:.3f} ms")


if __name__ == "__main__":
    main()
