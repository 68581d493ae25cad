"""Prompts and decode steps through a stack of 4-bit attention blocks over a paged cache.

    python examples/paged_decode.py [--cache float16|float8_e4m3fn|int8] [--layers 4] [--steps 32]

Every block is tilelang_amd.W4Attention: a fused W4A16 projection, rotation and cache write in one launch, attention of the new
tokens over the cache, the W4A16 projection back.  Weights are random; the first step's attention is compared with plain torch.
"""

from __future__ import annotations

import argparse
import os
import sys
import time

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import torch  # noqa: E402

import tilelang_amd as tl  # noqa: E402


def plain_attention(q, k, v):
    """One token's heads over its sequence, in fp32: q [heads, dim], k and v [tokens, kv_heads, dim]."""
    kv_heads, dim = k.shape[1:]
    q = q.float().view(kv_heads, -1, dim)
    scores = torch.softmax(q @ k.float().permute(1, 2, 0).contiguous() * dim**-0.5, dim=-1)
    return (scores @ v.float().transpose(0, 1).contiguous()).view(-1, dim)


def main() -> None:
    args = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    args.add_argument("--cache", default="float16", choices=("float16", "float8_e4m3fn", "int8"))
    args.add_argument("--layers", type=int, default=4)
    args.add_argument("--steps", type=int, default=32)
    args = args.parse_args()
    device, hidden, heads, kv_heads, dim, prompts = "cuda", 4096, 32, 8, 128, (200, 37, 512, 1)
    gen = torch.Generator().manual_seed(0)
    table = tl.rotary_table(4096, dim, device=device)
    layers = [tl.W4Attention(hidden, heads, kv_heads, dim, table).to(device) for _ in range(args.layers)]
    for layer in layers:
        for linear in (layer.qkv, layer.o):
            linear.load_float_weight(torch.randn((linear.out_features, linear.in_features), generator=gen) * linear.in_features**-0.5)
    cache = tl.PagedKVCache(len(prompts), pages=256, kv_heads=kv_heads, head_dim=dim, page_size=64, max_tokens=4096, layers=args.layers,
                            cache_dtype=None if args.cache == "float16" else args.cache, device=device)

    def step(x, counts):
        rows = cache.extend(counts)
        for i, layer in enumerate(layers):
            x = x + layer(x, cache, rows, i)
        return x

    x = step(torch.randn((sum(prompts), hidden), generator=gen).half().to(device), prompts)
    x = x[torch.tensor(prompts).cumsum(0).to(device) - 1]  # every sequence's last token goes on

    # the first block of the next step, by hand
    rows = cache.extend([1] * len(prompts))
    qkv = layers[0].qkv(x).view(len(prompts), heads + 2 * kv_heads, dim)
    got = layers[0].attend(qkv, cache, rows)
    q = tl.rotary(len(prompts), heads, dim, positions=table.shape[0])(qkv[:, :heads].contiguous(), table, rows.positions)
    keys, values = cache.read()
    starts = [0, *torch.tensor(cache.lengths).cumsum(0).tolist()]
    off = max((got[b].float() - plain_attention(q[b], keys[starts[b] : starts[b + 1]], values[starts[b] : starts[b + 1]])).abs().max().item()
              for b in range(len(prompts)))
    print(f"attention of the first step: largest difference from plain torch {off:.2e}")

    def steps(x, n):
        for _ in range(n):
            x = step(x, [1] * len(prompts))
            x = x / x.float().pow(2).mean(dim=-1, keepdim=True).sqrt().half()
        torch.cuda.synchronize()
        return x

    x = steps(x, 3)  # (the first of each kernel is loaded)
    began = time.perf_counter()
    x = steps(x, args.steps)
    spent = time.perf_counter() - began
    print(f"{args.steps} steps of {len(prompts)} sequences, {args.layers} blocks, {args.cache} cache: {spent / args.steps * 1e6:.0f} us a step, "
          f"lengths {cache.lengths}, finite: {bool(torch.isfinite(x).all())}")


if __name__ == "__main__":
    main()
