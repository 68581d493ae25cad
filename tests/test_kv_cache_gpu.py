"""The paged key-value cache as it is written (alone and with the rotation in the same launch) and read back."""

import math

import pytest
import torch

import tilelang_amd as tl
from kv_reference import HALF_ULP, TOP, fill_cache, rotate, stale, tokens_of

pytestmark = pytest.mark.gpu

DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float8_e4m3fn": torch.float8_e4m3fn, "int8": torch.int8}
SHAPES = [  # tokens, heads, kv_heads, head_dim, rotary_dim, interleaved, pages, page_size
    (1, 1, 1, 64, 64, False, 1, 8),
    (16, 32, 8, 128, 128, False, 5, 16),
    (37, 6, 3, 96, 48, True, 9, 64),
    (53, 5, 1, 112, 56, False, 7, 16),
    (23, 4, 4, 80, 32, False, 4, 32),
    (70, 2, 1, 256, 256, True, 2, 1024),
    (9, 3, 1, 72, 20, False, 3, 8),
    (1200, 8, 4, 128, 64, False, 90, 16),
]


def _empty_cache(pages, kv_heads, page_size, dim, held, device):
    raw = torch.full((pages, kv_heads, page_size, dim), 0x55, dtype=torch.uint8 if held.itemsize == 1 else torch.int16, device=device)
    scale = torch.full((pages, kv_heads, page_size), -7.0, device=device) if held.itemsize == 1 else None
    return raw.view(held), scale


def _spacing(z):
    """Distance of e4m3 values around z."""
    return torch.exp2(torch.floor(torch.log2(z.abs().clamp(min=2.0**-6))) - 3)


def _check_written(cache, scale, slots, x, slack, held):
    """x: exact values [tokens, kv_heads, head_dim] in 64 bits, slack the bound of what the kernel's fp32 may be off them."""
    pages, _, page_size, _ = cache.shape
    ok = (slots >= 0) & (slots < pages * page_size)
    page, place = (slots[ok] // page_size).long(), (slots[ok] % page_size).long()
    x, slack = x[ok], slack[ok]
    if held in TOP:
        codes = cache.view(torch.uint8)[page, :, place].view(held).double()
        s = scale[page, :, place].double()
        want = x.abs().amax(dim=-1) / TOP[held]
        # the largest magnitude's own error and a division
        assert ((s - want).abs() <= want * 2.0**-22 + slack.amax(dim=-1) / TOP[held]).all()
        z = torch.where(want[..., None] > 0, x / want[..., None], 0.0)
        step = torch.ones_like(z) if held == torch.int8 else _spacing(z)
        # to nearest, but for what fp32 is off: relative 2^-21 from two divisions and a product, and the value's own error
        off = step * 0.5 + z.abs() * 2.0**-21 + 2.5 * slack / want.clamp(min=1e-30)[..., None]
        assert ((codes - z).abs() <= off).all(), ((codes - z).abs() - off).max()
    else:
        got = cache[page, :, place].double()
        assert ((got - x).abs() <= HALF_ULP[held] * 1.01 * x.abs() + 1.01 * slack + 2.0**-25).all()
    # nothing else was touched
    raw = (cache.view(torch.uint8) if held.itemsize == 1 else cache.view(torch.int16)).clone()
    raw[page, :, place] = 0x55
    assert (raw == 0x55).all()
    if scale is not None:
        rest = scale.clone()
        rest[page, :, place] = -7.0
        assert (rest == -7.0).all()


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("cache", ["same", "float8_e4m3fn", "int8"])
@pytest.mark.parametrize("tokens,heads,kv_heads,dim,rotary_dim,interleaved,pages,page_size", SHAPES)
def test_write(cuda, tokens, heads, kv_heads, dim, rotary_dim, interleaved, pages, page_size, cache, dtype):
    print(f"write {tokens} {heads}/{kv_heads}x{dim} r={rotary_dim} {interleaved} {pages}x{page_size} {cache} {dtype}", flush=True)
    held = DTYPES[dtype if cache == "same" else cache]
    gen = torch.Generator().manual_seed(tokens * 3 + dim)
    qkv = torch.randn((tokens, heads + 2 * kv_heads, dim), generator=gen).to(DTYPES[dtype]).to(cuda)
    order = torch.randperm(pages * page_size, generator=gen)
    slots = torch.full((tokens,), -1, dtype=torch.int32)
    n = min(tokens, pages * page_size)
    slots[:n] = order[:n].int()
    if tokens > 4:  # places of the batch that hold no token
        slots[1], slots[3] = -1, pages * page_size
    slots = slots.to(cuda)
    rows = 2000
    table = tl.rotary_table(rows, rotary_dim, device=cuda)
    positions = torch.randint(0, rows, (tokens,), generator=gen, dtype=torch.int32).to(cuda)
    pool = dict(kv_heads=kv_heads, head_dim=dim, pages=pages, page_size=page_size, dtype=dtype, cache_dtype=None if cache == "same" else cache)

    (kc, ks), (vc, vs) = (_empty_cache(pages, kv_heads, page_size, dim, held, cuda) for _ in range(2))
    buffers = (kc, vc) if ks is None else (kc, vc, ks, vs)
    q = tl.rotary_kv_cache_write(tokens, heads, positions=rows, rotary_dim=rotary_dim, interleaved=interleaved, **pool)(
        qkv, table, positions, slots, *buffers)
    want, slack = rotate(qkv[:, : heads + kv_heads], table, positions, rotary_dim, interleaved)
    assert ((q.double() - want[:, :heads]).abs() <= HALF_ULP[q.dtype] * 1.01 * want[:, :heads].abs() + 1.01 * slack[:, :heads] + 2.0**-25).all()
    _check_written(kc, ks, slots, want[:, heads:], slack[:, heads:], held)
    v = qkv[:, heads + kv_heads :].double()
    _check_written(vc, vs, slots, v, torch.zeros_like(v), held)

    # without the rotation, keys and values apart
    (kc, ks), (vc, vs) = (_empty_cache(pages, kv_heads, page_size, dim, held, cuda) for _ in range(2))
    k = qkv[:, :kv_heads].contiguous()
    buffers = (kc, vc) if ks is None else (kc, vc, ks, vs)
    assert tl.kv_cache_write(tokens, **pool)(k, qkv[:, heads + kv_heads :].contiguous(), slots, *buffers) is None
    _check_written(kc, ks, slots, k.double(), torch.zeros_like(k.double()), held)
    _check_written(vc, vs, slots, v, torch.zeros_like(v), held)


@pytest.mark.parametrize("cache", ["float8_e4m3fn", "int8"])
def test_odd_rows(cuda, cache):
    """Zeros, the smallest and largest numbers, one large among small ones, infinities and NaN; the row beside each stays."""
    dim, kv_heads, page_size = 64, 2, 8
    x = torch.randn((8, kv_heads, dim), generator=torch.Generator().manual_seed(2)).bfloat16()
    x[0, 0] = 0
    x[1, 0] = 1e-35
    x[2, 0] *= 2.0**-90
    x[3, 0, 5] = 3e38
    x[4, 0, 63] = math.inf
    x[5, 0, 0] = math.nan
    x[6, 0, 9] = -math.inf
    x[7, 0] = -2.0**-120
    x = x.to(cuda)
    held = DTYPES[cache]
    (kc, ks), (vc, vs) = (_empty_cache(1, kv_heads, page_size, dim, held, cuda) for _ in range(2))
    pool = dict(kv_heads=kv_heads, head_dim=dim, pages=1, page_size=page_size, dtype="bfloat16", cache_dtype=cache)
    slots = torch.arange(8, dtype=torch.int32, device=cuda)
    tl.kv_cache_write(8, **pool)(x, x, slots, kc, vc, ks, vs)
    table, starts = torch.zeros((1, 1), dtype=torch.int32, device=cuda), torch.tensor([0, 8], dtype=torch.int32, device=cuda)
    k, v = tl.kv_cache_read(1, 8, max_pages=1, **pool)(kc, vc, ks, vs, table, starts)
    assert torch.equal(k.nan_to_num(9.0), v.nan_to_num(9.0))
    assert torch.isnan(k[[4, 5, 6], 0]).all() and not torch.isnan(k[[0, 1, 2, 3, 7], 0]).any() and not torch.isnan(k[:, 1]).any()
    assert (k[[0, 1, 7], 0] == 0).all() and (ks[0, 0, [0, 1, 7]] == 0).all()
    step = 2.0**-3 if cache == "float8_e4m3fn" else 1 / 127
    most = x[[2, 3], 0].float().abs().amax(dim=-1, keepdim=True)
    assert ((k[[2, 3], 0].float() - x[[2, 3], 0].float()).abs() <= most * step).all()
    assert (k[2, 0] != 0).any() and k[3, 0, 5] > 2.9e38


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("cache", ["same", "float8_e4m3fn", "int8"])
@pytest.mark.parametrize("lengths,kv_heads,dim,page_size,extra", [
    ([1], 1, 64, 8, 0), ([0, 5, 0, 0, 40, 17, 0], 3, 80, 16, 0), ([100, 33], 8, 128, 32, 5), ([7, 8, 9, 1000, 1], 2, 256, 8, 0),
    ([1030], 5, 96, 1024, 3), ([3] * 200, 1, 72, 8, 0),
])
def test_read(cuda, lengths, kv_heads, dim, page_size, extra, cache, dtype):
    print(f"read {lengths[:8]} {kv_heads}x{dim} page {page_size} {cache} {dtype}", flush=True)
    held = DTYPES[dtype if cache == "same" else cache]
    gen = torch.Generator().manual_seed(sum(lengths) + dim)
    counts = [-(-n // page_size) for n in lengths]
    pages, width = sum(counts) + 2, max(counts) + 1
    order = torch.randperm(pages, generator=gen).int()
    table = torch.full((len(lengths), width), -5, dtype=torch.int32)
    for b, n in enumerate(counts):
        table[b, :n] = order[sum(counts[:b]) : sum(counts[: b + 1])]
    missing = max(range(len(lengths)), key=lambda b: lengths[b])
    if counts[missing] > 1:  # a page that is not there
        table[missing, 1] = pages
    buffers = []
    for _ in range(2):
        c, s = fill_cache(gen, pages, kv_heads, page_size, dim, held, cuda)
        for b, n in enumerate(lengths):
            if n % page_size:
                stale(c, s, int(table[b, n // page_size]) if table[b, n // page_size] < pages else int(order[-1]), n % page_size)
        buffers.append((c, s))
    (kc, ks), (vc, vs) = buffers
    starts = torch.tensor([0] + lengths).cumsum(0).int()
    tokens = int(starts[-1]) + extra
    kernel = tl.kv_cache_read(len(lengths), tokens, kv_heads, dim, pages, page_size, width, dtype=dtype, cache_dtype=None if cache == "same" else cache)
    got = kernel(*((kc, vc) if ks is None else (kc, vc, ks, vs)), table.to(cuda), starts.to(cuda))
    assert got.shape == (2, tokens, kv_heads, dim)
    for which, (c, s) in enumerate(buffers):
        want = torch.cat([tokens_of(c, s, table[b], n) for b, n in enumerate(lengths)] + [torch.zeros((extra, kv_heads, dim), dtype=torch.float64)])
        absent = torch.isnan(want)
        assert not (absent & (torch.arange(tokens)[:, None, None] >= int(starts[-1]))).any()
        # a product in fp32 and the result's rounding
        off = (got[which].cpu().double() - want.nan_to_num(0.0)).abs()
        assert (off <= (HALF_ULP[got.dtype] + 2.0**-23) * want.nan_to_num(0.0).abs() + 2.0**-25).all()


def test_write_then_read_keeps_sixteen_bits(cuda):
    """Through a cache of the activations' own type every bit comes back, NaN and infinities among them."""
    tokens, kv_heads, dim, page_size, pages = 130, 4, 128, 16, 12
    x = torch.randint(-(2**15), 2**15, (2, tokens, kv_heads, dim), generator=torch.Generator().manual_seed(1), dtype=torch.int16).to(cuda)
    x &= torch.tensor(-2, dtype=torch.int16, device=cuda)  # (a quiet NaN stays what it is; the payload's last bit is not looked at)
    x = torch.where((x & 0x7C00) == 0x7C00, x | 0x0200, x)
    k, v = x.view(torch.float16)
    pool = dict(kv_heads=kv_heads, head_dim=dim, pages=pages, page_size=page_size)
    kc, vc = (torch.zeros((pages, kv_heads, page_size, dim), dtype=torch.float16, device=cuda) for _ in range(2))
    table = torch.randperm(pages, generator=torch.Generator().manual_seed(4)).int()[None].to(cuda)
    at = torch.arange(tokens, device=cuda)
    slots = (table[0, at // page_size] * page_size + at % page_size).int()
    tl.kv_cache_write(tokens, **pool)(k.contiguous(), v.contiguous(), slots, kc, vc)
    got = tl.kv_cache_read(1, tokens, max_pages=pages, **pool)(kc, vc, table, torch.tensor([0, tokens], dtype=torch.int32, device=cuda))
    assert torch.equal(got.view(torch.int16), x)
