"""PagedKVCache and W4Attention: the bookkeeping of pages on the CPU; on the GPU prompts and decode steps against the formulas on
what the layer has in hand."""

import pytest
import torch

import tilelang_amd as tl
from kv_reference import attention, attention_bound, tokens_of


def _cache(**more):
    return tl.PagedKVCache(**(dict(sequences=3, pages=6, kv_heads=2, head_dim=64, page_size=8, device="cpu") | more))


def test_pages_as_sequences_grow():
    cache = _cache(max_tokens=24)
    rows = cache.extend([9, 0, 1])
    assert cache.lengths == [9, 0, 1] and rows.positions.tolist() == [*range(9), 0] and rows.lengths.tolist() == [*range(1, 10), 1]
    used = cache.page_table[cache.page_table >= 0].tolist()
    assert len(used) == len(set(used)) == 3 and (cache.page_table[1] == -1).all()
    for r, (b, t) in enumerate([(0, t) for t in range(9)] + [(2, 0)]):
        assert rows.slots[r] == int(cache.page_table[b, t // 8]) * 8 + t % 8 and torch.equal(rows.pages[r], cache.page_table[b])
    step = cache.extend([1, 1, 1])
    assert step.pages is cache.page_table and step.positions.tolist() == [9, 0, 1] and step.lengths.tolist() == [10, 1, 2]
    with pytest.raises(RuntimeError, match="3 pages wanted, 2 free"):
        cache.extend([7, 8, 7])  # takes nothing
    assert cache.lengths == [10, 1, 2] and (cache.page_table >= 0).sum() == 4
    with pytest.raises(RuntimeError, match="max_tokens=24"):
        cache.extend([15, 0, 0])
    cache.release(0)
    assert cache.lengths == [0, 1, 2] and (cache.page_table[0] == -1).all()
    cache.extend([0, 23, 0])  # the pages of the one that went
    used = cache.page_table[cache.page_table >= 0].tolist()
    assert len(used) == len(set(used)) == 4
    with pytest.raises(ValueError, match="3 counts"):
        cache.extend([1, 1])
    with pytest.raises(ValueError, match="some positive"):
        cache.extend([0, 0, 0])


@pytest.mark.parametrize("changed,match", [(dict(page_size=12), "page_size=12"), (dict(cache_dtype="bfloat16"), "cache_dtype"), (dict(sequences=0), "sequences"),
                                           (dict(layers=0), "layers"), (dict(max_tokens=0), "max_tokens")])
def test_cache_refuses(changed, match):
    with pytest.raises(ValueError, match=match):
        _cache(**changed)


def test_read_of_no_tokens():
    k, v = _cache().read()
    assert k.shape == v.shape == (0, 2, 64) and k.dtype == torch.float16


@pytest.mark.gpu
@pytest.mark.parametrize("held", [None, "float8_e4m3fn", "int8"])
@pytest.mark.parametrize("interleaved,window,sinks,dim,rotary_dim", [(False, 0, False, 64, 64), (True, 20, True, 128, 32)])
def test_prompts_and_steps(cuda, held, interleaved, window, sinks, dim, rotary_dim):
    print(f"layer {held} interleaved {interleaved} window {window} sinks {sinks} {dim} {rotary_dim}", flush=True)
    hidden, heads, kv_heads, layers = 256, 8, 2, 2
    gen = torch.Generator().manual_seed(dim)
    table = tl.rotary_table(300, rotary_dim, device=cuda)
    blocks = [tl.W4Attention(hidden, heads, kv_heads, dim, table, interleaved=interleaved, window=window, sinks=sinks).to(cuda) for _ in range(layers)]
    for block in blocks:
        for linear in (block.qkv, block.o):
            linear.load_float_weight(torch.randn((linear.out_features, linear.in_features), generator=gen) * 0.1)
        if sinks:
            block.sinks.copy_(torch.randn(heads, generator=gen))
    cache = tl.PagedKVCache(4, pages=40, kv_heads=kv_heads, head_dim=dim, page_size=16, max_tokens=300, layers=layers, cache_dtype=held, device=cuda)
    for counts in ([70, 5, 0, 33], [1, 1, 1, 1], [3, 0, 40, 1], [1, 1, 1, 1]):
        rows = cache.extend(counts)
        x = torch.randn((sum(counts), hidden), generator=gen).half().to(cuda)
        owners = [b for b, c in enumerate(counts) for _ in range(c)]
        for i, block in enumerate(blocks):
            qkv = block.qkv(x).view(len(owners), heads + 2 * kv_heads, dim)
            got = block.attend(qkv, cache, rows, i)
            # (the whole layer: the same, and projected back)
            assert torch.equal(block(x, cache, rows, i), block.o(got.reshape(len(owners), -1)))
            turned = tl.rotary(len(owners), heads, dim, positions=300, rotary_dim=rotary_dim, interleaved=interleaved,
                               row_stride=(heads + 2 * kv_heads) * dim)(qkv[:, :heads], table, rows.positions)
            pool = cache.pool(i)
            for r in range(0, len(owners), 7):
                n = int(rows.lengths[r])
                k, v = (tokens_of(pool[w], None if held is None else pool[2 + w], cache.page_table[owners[r]], n) for w in range(2))
                want, _, spread = attention(turned[r], k, v, dim**-0.5, window, block.sinks.cpu() if sinks else None)
                off = (got[r].cpu().double() - want).abs()
                assert (off <= attention_bound(want, spread, got.dtype, cache.cache_dtype)).all(), (counts, r)
            x = block.o(got.reshape(len(owners), -1))
    keys, values = cache.read(1)
    at = 0
    for b, n in enumerate(cache.lengths):
        for got, w in ((keys, 0), (values, 1)):
            want = tokens_of(cache.pool(1)[w], None if held is None else cache.pool(1)[2 + w], cache.page_table[b], n)
            assert ((got[at : at + n].cpu().double() - want).abs() <= 2.0**-11 * 1.01 * want.abs() + 2.0**-25).all()
        at += n
    assert at == sum(cache.lengths) == keys.shape[0]
