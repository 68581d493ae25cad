"""What the rotation, the cache and the attention over it promise, refuse and keep, without a GPU."""

import math
import os

import pytest
import torch

import tilelang_amd as tl
from tilelang_amd.kv_kernels import attention_sequences

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


@pytest.mark.parametrize("heads,kv_heads,page_size,max_pages", [(32, 8, 16, 4), (64, 8, 16, 8192), (33, 1, 1024, 2**20), (128, 128, 64, 2**14), (4096, 4096, 8, 1)])
def test_sequences_of_a_call(heads, kv_heads, page_size, max_pages):
    """The factory refuses what the entry point would refuse at the launch, and no more.  (A scale of NaN, which is looked at after the
    sequences, keeps the entry point from launching.)"""
    from test_kv_host import _entry

    most = attention_sequences(heads, kv_heads, page_size * max_pages)
    sizes = dict(heads=heads, kv_heads=kv_heads, page_size=page_size, max_pages=max_pages)
    for n, match in ((most, "scale must be finite"), (most + 1, "at most 65535" if most == 65535 else "the work that a call counts")):
        rc, message = _entry("call_paged_attention_decode", sequences=n, scale=math.nan, **sizes)
        assert rc == -1 and match in message, (n, message)
    tl.paged_attention_decode(most, head_dim=64, pages=2, **sizes)
    with pytest.raises(ValueError, match=f"at most {most} sequences"):
        tl.paged_attention_decode(most + 1, head_dim=64, pages=2, **sizes)


@pytest.mark.parametrize("make", [
    lambda n: tl.rotary(n, 8, 64, positions=5),
    lambda n: tl.kv_cache_write(n, kv_heads=4, head_dim=64, pages=3, page_size=16),
    lambda n: tl.rotary_kv_cache_write(n, 4, positions=5, kv_heads=2, head_dim=64, pages=3, page_size=16),
    lambda n: tl.kv_cache_read(1, n, kv_heads=8, head_dim=64, pages=3, page_size=16, max_pages=2),
])
def test_heads_of_a_call(make):
    make(2**22)
    with pytest.raises(ValueError, match="at most 33554432 heads"):
        make(2**22 + 1)


def test_a_prompt_of_many_rows(monkeypatch):
    """Its page table is not copied for every row, and the layer goes through it in parts that the library takes, each one written before
    it is attended to, and before the next."""
    cache = tl.PagedKVCache(2, pages=5000, kv_heads=1, head_dim=64, page_size=16, max_tokens=70000, device="cpu")
    rows = cache.extend([69000, 1000])
    assert rows.pages is cache.page_table and rows.owners.tolist() == [0] * 69000 + [1] * 1000
    assert torch.equal(rows.pages_of(slice(68999, 69002)), cache.page_table[[0, 1, 1]])
    layer = tl.W4Attention(128, 4, 1, 64, tl.rotary_table(70000, 64))
    seen = []

    def kernel(make, n, *_, **__):
        def call(first, *operands):
            pages, lengths = operands[-2:]
            seen.append((make.__name__, n, int(operands[1][0] if make is tl.rotary_kv_cache_write else lengths[0] - 1)))
            if make is tl.paged_attention_decode:
                assert pages.shape == (n, cache.max_pages) and lengths.shape == (n,)
            return first[:, :4].contiguous()

        return call

    monkeypatch.setattr(cache, "kernel", kernel)
    qkv = torch.arange(70000.0)[:, None, None].expand(70000, 6, 64)
    assert torch.equal(layer.attend(qkv, cache, rows), qkv[:, :4])
    most = layer._rows_at_once(cache)
    assert most * cache.max_pages <= 2**26 and most < 65536
    starts = range(0, 70000, most)
    assert seen == [(name, min(most, 70000 - at), at if at < 69000 else at - 69000) for at in starts for name in ("rotary_kv_cache_write", "paged_attention_decode")]


def test_rows_keep_their_pages():
    """What a step was given stays as it was when a sequence grows or goes, one token a sequence or several."""
    cache = tl.PagedKVCache(2, pages=20, kv_heads=1, head_dim=64, page_size=8, max_tokens=64, device="cpu")
    for counts in ([7, 8], [1, 1], [1, 1], [3, 0], [20, 20]):
        rows, table = cache.extend(counts), cache.page_table.tolist()
        owners = [b for b, c in enumerate(counts) for _ in range(c)]
        kept = rows.pages.tolist()
        assert kept == [table[b] for b in owners]
        cache.extend([8, 8])
        assert rows.pages.tolist() == kept
        for b in range(2):
            cache.release(b)
        assert rows.pages.tolist() == kept and (cache.page_table == -1).all()


def test_kernels_that_a_cache_keeps():
    """Not one for every number of rows that there ever was; those in use stay."""
    cache = tl.PagedKVCache(1, pages=2, kv_heads=2, head_dim=64, page_size=8, device="cpu")
    step = cache.kernel(tl.kv_cache_write, 1)
    for n in range(2, 1000):
        prompt = cache.kernel(tl.kv_cache_write, n)
        assert prompt.params[0].shape[0] == n and cache.kernel(tl.kv_cache_write, n) is prompt
        assert cache.kernel(tl.kv_cache_write, 1) is step
    assert len(cache._kernels) == 64


@pytest.mark.parametrize("turned", [lambda m: m.half(), lambda m: m.bfloat16(), lambda m: m.to(torch.float16), lambda m: m.double(), lambda m: m.half().float()])
def test_table_and_sinks_stay_in_32_bits(turned):
    """A model is turned into another type as a whole; its positions' table and its sinks are not."""
    table = tl.rotary_table(50000, 64)
    layer = tl.W4Attention(128, 4, 1, 64, table, sinks=True)
    layer.sinks.copy_(torch.randn(4, generator=torch.Generator().manual_seed(0)))
    sinks = layer.sinks.clone()
    model = torch.nn.Sequential(layer, torch.nn.Linear(8, 8))
    turned(model)
    assert layer.rotary.dtype == layer.sinks.dtype == torch.float32
    assert torch.equal(layer.rotary, table) and torch.equal(layer.sinks, sinks)
    assert layer.to("meta").rotary.device.type == "meta"


def test_table_and_sinks_where_there_are_none():
    layer = tl.W4Attention(128, 4, 1, 64, tl.rotary_table(10, 64)).half()
    assert layer.sinks is None and layer.rotary.dtype == torch.float32
