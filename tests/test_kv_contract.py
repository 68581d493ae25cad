"""What the rotation, the cache and the attention over it promise, refuse and keep, without a GPU."""

import os

import pytest
import torch

import tilelang_amd as tl

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_slots_of_a_call_are_distinct():
    """Rows are written by independent lanes, codes and scale by stores of their own: no entry point promises anything for a place that two
    tokens name, and the cache's own bookkeeping never names one twice."""
    with open(os.path.join(ROOT, "include", "dqgemm.h")) as f:
        header = f.read()
    assert "same slot: one of them" not in header and "slots of a call have to be distinct" in header
    for factory in (tl.kv_cache_write, tl.rotary_kv_cache_write):
        assert "distinct" in factory.__doc__
    cache = tl.PagedKVCache(4, pages=40, kv_heads=1, head_dim=64, page_size=8, device="cpu")
    held = [[] for _ in range(4)]
    for counts in ([9, 0, 1, 30], [1, 1, 1, 1], [0, 20, 7, 0], [1, 1, 1, 1], [8, 8, 8, 8]):
        slots = cache.extend(counts).slots.tolist()
        for b, c in enumerate(counts):
            held[b] += slots[:c]
            slots = slots[c:]
        everything = [s for sequence in held for s in sequence]
        assert len(set(everything)) == len(everything)
        if len(held[2]) > 20:
            cache.release(3)
            held[3] = []


@pytest.mark.parametrize("make", [
    lambda: tl.rotary(2, 2, 64, positions=5, row_stride=2**32 + 128),
    lambda: tl.rotary(2, 2, 64, positions=2**32 + 5),
    lambda: tl.rotary(2**32 + 1, 2, 64, positions=5),
    lambda: tl.kv_cache_write(2**32 + 1, kv_heads=2, head_dim=64, pages=3, page_size=16),
    lambda: tl.kv_cache_write(1, kv_heads=2**32 + 2, head_dim=64, pages=3, page_size=16),
    lambda: tl.rotary_kv_cache_write(1, 2**32 + 4, positions=5, kv_heads=2, head_dim=64, pages=3, page_size=16),
    lambda: tl.kv_cache_read(1, 2**32 + 9, kv_heads=2, head_dim=64, pages=3, page_size=16, max_pages=2),
    lambda: tl.kv_cache_read(1, 9, kv_heads=2, head_dim=64, pages=3, page_size=16, max_pages=2**32 + 2),
])
def test_sizes_beyond_32_bits(make):
    """Refused, and not taken by their lower 32 bits."""
    with pytest.raises(ValueError, match="32-bit"):
        make()
