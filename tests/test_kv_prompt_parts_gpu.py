"""A prompt that the layer takes in parts, against the same prompt in one."""

import pytest
import torch

import tilelang_amd as tl
from tilelang_amd import attention
from kv_reference import attention_bound, tokens_of
from kv_reference import attention as exact

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("held", [None, "int8"])
def test_parts_of_a_prompt(cuda, held, monkeypatch):
    hidden, heads, kv_heads, dim, counts = 256, 8, 2, 64, [150, 0, 77]
    gen = torch.Generator().manual_seed(4)
    block = tl.W4Attention(hidden, heads, kv_heads, dim, tl.rotary_table(200, dim, device=cuda)).to(cuda)
    for linear in (block.qkv, block.o):
        linear.load_float_weight(torch.randn((linear.out_features, linear.in_features), generator=gen) * 0.1)
    x = torch.randn((sum(counts), hidden), generator=gen).half().to(cuda)
    qkv = block.qkv(x).view(-1, heads + 2 * kv_heads, dim)

    def run():
        cache = tl.PagedKVCache(3, pages=40, kv_heads=kv_heads, head_dim=dim, page_size=16, max_tokens=200, cache_dtype=held, device=cuda)
        rows = cache.extend(counts)
        return cache, rows, block.attend(qkv, cache, rows)

    _, whole_rows, whole = run()
    assert whole_rows.owners is None
    monkeypatch.setattr(attention, "MAX_PAGE_IDS", 40 * 13)  # 40 rows of 13 pages
    cache, rows, parts = run()
    assert rows.owners is not None and block._rows_at_once(cache) == 40 and parts.shape == whole.shape
    owners = [b for b, c in enumerate(counts) for _ in range(c)]
    q = tl.rotary(sum(counts), heads, dim, positions=200, row_stride=(heads + 2 * kv_heads) * dim)(qkv[:, :heads], block.rotary, rows.positions)
    for r in range(0, len(owners), 3):
        pool = cache.pool()
        k, v = (tokens_of(pool[w], None if held is None else pool[2 + w], cache.page_table[owners[r]], int(rows.lengths[r])) for w in range(2))
        want, _, spread = exact(q[r], k, v, dim**-0.5)
        for got in (whole, parts):
            assert ((got[r].cpu().double() - want).abs() <= attention_bound(want, spread, got.dtype, cache.cache_dtype)).all(), r
