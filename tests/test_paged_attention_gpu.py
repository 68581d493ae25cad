"""Attention of one new token over the paged cache against the formula in 64 bits, over lengths, heads, types, windows and sinks."""

import math

import pytest
import torch

import tilelang_amd as tl
from kv_reference import attention, attention_bound, fill_cache, stale, tokens_of

pytestmark = pytest.mark.gpu

DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float8_e4m3fn": torch.float8_e4m3fn, "int8": torch.int8}


class _Case:
    def __init__(self, cuda, lengths, heads, kv_heads, dim, page_size, dtype, cache="same", wide=2, seed=0, q_scale=2.0):
        self.held = DTYPES[dtype if cache == "same" else cache]
        gen = torch.Generator().manual_seed(seed + sum(lengths) + heads * dim)
        self.lengths, self.heads = lengths, heads
        counts = [-(-n // page_size) for n in lengths]
        self.pages, width = sum(counts) + 2, max(counts) + wide
        order = torch.randperm(self.pages, generator=gen).int()
        self.table = torch.full((len(lengths), width), -1, dtype=torch.int32)
        for b, n in enumerate(counts):
            self.table[b, :n] = order[sum(counts[:b]) : sum(counts[: b + 1])]
        self.buffers = []
        for _ in range(2):
            c, s = fill_cache(gen, self.pages, kv_heads, page_size, dim, self.held, cuda)
            for b, n in enumerate(lengths):
                if n % page_size:
                    stale(c, s, int(self.table[b, n // page_size]), n % page_size)
            self.buffers.append((c, s))
        self.q = (torch.randn((len(lengths), heads, dim), generator=gen) * q_scale).to(DTYPES[dtype]).to(cuda)
        self.sinks = torch.randn((heads,), generator=gen).to(cuda)
        self.sizes = dict(kv_heads=kv_heads, head_dim=dim, pages=self.pages, page_size=page_size, max_pages=width, dtype=dtype,
                          cache_dtype=None if cache == "same" else cache)
        self.dim, self.device = dim, cuda

    def pool(self):
        (kc, ks), (vc, vs) = self.buffers
        return (kc, vc) if ks is None else (kc, vc, ks, vs)

    def run(self, window=0, sinks=False, scale=None, lengths=None):
        n = torch.tensor(self.lengths if lengths is None else lengths, dtype=torch.int32, device=self.device)
        kernel = tl.paged_attention_decode(len(self.lengths), self.heads, window=window, sinks=sinks, scale=scale, with_lse=True, **self.sizes)
        return kernel(self.q, *self.pool(), self.table.to(self.device), n, *((self.sinks,) if sinks else ()))

    def check(self, window=0, sinks=False, scale=None, there=None):
        out, lse = self.run(window, sinks, scale)
        assert not torch.isnan(out).any()
        for b, n in enumerate(self.lengths):
            k, v = (tokens_of(c, s, self.table[b], n) for c, s in self.buffers)
            want, want_lse, spread = attention(self.q[b], k, v, self.dim**-0.5 if scale is None else scale, window,
                                               self.sinks.cpu() if sinks else None, there=None if there is None else there[b])
            off = (out[b].cpu().double() - want).abs()
            limit = attention_bound(want, spread, out.dtype, self.held)
            assert (off <= limit).all(), (b, n, (off / limit).max())
            # fp32 scores and sums
            near = (lse[b].cpu().double() - want_lse).abs() <= 2.0**-16 * (1 + want_lse.abs())
            assert (near | (lse[b].cpu().double() == want_lse)).all(), (b, lse[b], want_lse)


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("cache", ["same", "float8_e4m3fn", "int8"])
@pytest.mark.parametrize("lengths,heads,kv_heads,dim,page_size", [
    ([1], 1, 1, 64, 8),
    ([1, 2, 7, 8, 9, 0, 31, 32, 33], 4, 2, 64, 8),
    ([127, 128, 129, 500], 32, 8, 128, 16),
    ([1000], 8, 1, 80, 16),
    ([65, 300], 12, 12, 96, 64),
    ([44, 1], 34, 2, 112, 32),       # 17 heads share one: a second block of one head
    ([700, 3], 32, 1, 160, 128),
    ([260, 0, 19], 6, 2, 192, 16),
    ([515, 130], 16, 2, 256, 1024),
    ([5000, 40], 7, 1, 128, 32),
    ([77, 4, 5, 300], 16, 2, 64, 16),  # eight heads share one, and nine
    ([90, 700], 20, 1, 256, 16), ([33, 500, 0], 50, 2, 192, 32), ([77, 300], 18, 2, 64, 16), ([36, 1000], 8, 1, 112, 32), ([12, 640], 9, 1, 96, 8),
])
def test_lengths_heads_types(cuda, lengths, heads, kv_heads, dim, page_size, cache, dtype):
    print(f"attention {lengths} {heads}/{kv_heads}x{dim} page {page_size} {cache} {dtype}", flush=True)
    _Case(cuda, lengths, heads, kv_heads, dim, page_size, dtype, cache).check()


@pytest.mark.parametrize("cache", ["same", "float8_e4m3fn", "int8"])
@pytest.mark.parametrize("window,sinks", [(1, False), (5, True), (32, False), (100, True), (128, False), (0, True), (10000, True)])
def test_window_and_sinks(cuda, window, sinks, cache):
    case = _Case(cuda, [0, 1, 5, 31, 100, 129, 1111, 640], 16, 4, 64, 16, "bfloat16", cache)
    case.check(window=window, sinks=sinks)
    if not sinks:
        return
    out, lse = case.run(window, True)
    assert (out[0] == 0).all() and torch.allclose(lse[0], case.sinks, rtol=1e-6, atol=1e-6)


@pytest.mark.parametrize("cache", ["same", "int8"])
def test_empty_sequences_only(cuda, cache):
    case = _Case(cuda, [0, 0, 0], 8, 2, 128, 16, "float16", cache)
    out, lse = case.run()
    assert (out == 0).all() and (lse == -math.inf).all()


@pytest.mark.parametrize("cache", ["same", "float8_e4m3fn"])
def test_pages_that_are_not_there(cuda, cache):
    """Tokens of a page id outside of the cache count as absent, whole tiles and sequences of them too."""
    case = _Case(cuda, [500, 64, 200], 8, 2, 128, 16, "bfloat16", cache)
    there = [torch.ones(n, dtype=torch.bool) for n in case.lengths]
    for b, column, bad in ((0, 0, -1), (0, 7, case.pages), (0, 8, 2**31 - 1), (0, 9, -(2**31)), (0, 31, -1), (2, 3, case.pages)):
        case.table[b, column] = bad
        there[b][16 * column : 16 * column + 16] = False
    case.table[1] = -1
    there[1][:] = False
    case.check(there=there)
    case.check(there=there, window=40, sinks=True)


def test_lengths_beyond_the_table(cuda):
    """A length counts up to what the table's pages hold, and not below none."""
    case = _Case(cuda, [64, 64], 4, 4, 64, 16, "float16", wide=0)
    want, _ = case.run()
    got, lse = case.run(lengths=[2**31 - 1, -3])
    assert torch.equal(got[0], want[0]) and (got[1] == 0).all() and (lse[1] == -math.inf).all()


@pytest.mark.parametrize("dtype,cache", [("float16", "same"), ("bfloat16", "same"), ("bfloat16", "int8"), ("float16", "float8_e4m3fn")])
def test_peaked_and_growing_scores(cuda, dtype, cache):
    """Scores of some tens, largest last, so that the running maximum grows all the way; and one scale for equal weights."""
    case = _Case(cuda, [900], 8, 2, 64, 16, dtype, cache, q_scale=0.1)
    for (c, _) in case.buffers[:1]:
        pages = case.table[0, : 900 // 16 + 1].long().to(cuda)
        rising = torch.linspace(-1, 1, 16 * len(pages), device=cuda).reshape(len(pages), 1, 16, 1)
        if c.dtype == torch.int8:
            c[pages] = (rising * 127).round().to(torch.int8).expand_as(c[pages])
        elif c.dtype == torch.float8_e4m3fn:
            c.view(torch.uint8)[pages] = (rising * 400).to(c.dtype).view(torch.uint8).expand(len(pages), c.shape[1], 16, c.shape[3])
        else:
            c[pages] = rising.to(c.dtype).expand_as(c[pages])
    case.q.fill_(1.0)
    case.check(scale=0.5 if case.buffers[0][1] is None else 0.25)
    case.check(scale=0.0)


@pytest.mark.parametrize("cache", ["float8_e4m3fn", "int8"])
def test_scales_of_every_size(cuda, cache):
    """Tokens' scales over 2^-40 .. 2^20 and zero, and queries of bf16's range."""
    case = _Case(cuda, [333], 4, 1, 128, 16, "bfloat16", cache)
    gen = torch.Generator().manual_seed(7)
    (kc, ks), (vc, vs) = case.buffers
    live = ~torch.isnan(vs)
    vs[live] = torch.exp2(torch.randint(-40, 20, (int(live.sum()),), generator=gen).float()).to(cuda)
    vs[live & (torch.rand(vs.shape, generator=gen) < 0.1).to(cuda)] = 0.0
    case.check()
    case.q.mul_(2.0**100)
    case.check(scale=case.dim**-0.5 * 2.0**-100)
    case.q.mul_(2.0**-120).mul_(2.0**-60)
    case.check(scale=case.dim**-0.5 * 2.0**80)


def test_infinities_and_nan_that_live(cuda):
    """What a live token holds shows: a NaN value in its head's result, and nowhere else."""
    case = _Case(cuda, [100, 100], 4, 2, 64, 16, "float16")
    case.buffers[1][0][int(case.table[0, 2]), 1, 3, 9] = math.nan
    out, _ = case.run()
    assert torch.isnan(out[0, 2:, 9]).all()
    out[0, 2:, 9] = 0
    assert not torch.isnan(out).any()
    case.buffers[0][0][int(case.table[1, 0]), 0, 3, 9] = math.nan
    out, lse = case.run()
    assert torch.isnan(out[1, :2]).all() and torch.isnan(lse[1, :2]).all() and not torch.isnan(out[1, 2:]).any()


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_infinite_values(cuda, dtype):
    """An infinity among a head's values is one in its result, in that element alone; two of both signs are no number."""
    case = _Case(cuda, [100, 2000], 4, 2, 64, 16, dtype)
    values = case.buffers[1][0]
    values[int(case.table[0, 2]), 1, 3, 9] = math.inf
    values[int(case.table[1, 5]), 0, 3, 7] = -math.inf
    values[int(case.table[1, 90]), 0, 1, 8], values[int(case.table[1, 3]), 0, 1, 8] = math.inf, -math.inf
    out, lse = case.run()
    assert (out[0, 2:, 9] == math.inf).all() and (out[1, :2, 7] == -math.inf).all() and torch.isnan(out[1, :2, 8]).all()
    out[0, 2:, 9] = out[1, :2, 7] = out[1, :2, 8] = 0
    assert torch.isfinite(out).all() and torch.isfinite(lse).all()


@pytest.mark.parametrize("cache", ["same", "int8"])
def test_parts_join(cuda, cache):
    """Results over a context's first and second half, joined by their logarithms, are those over the whole."""
    case = _Case(cuda, [640], 8, 2, 128, 16, "float16", cache)
    whole, lse = case.run()
    n = 20
    parts = []
    for columns in (slice(0, n), slice(n, 40)):
        keep = case.table.clone()
        case.table = torch.cat([keep[:, columns], torch.full((1, keep.shape[1] - n), -1, dtype=torch.int32)], dim=1)
        parts.append(case.run(lengths=[320]))
        case.table = keep
    both = torch.stack([p[1] for p in parts])
    weights = torch.softmax(both.double(), dim=0)
    joined = sum(w[..., None] * p[0].double() for w, p in zip(weights, parts))
    assert torch.allclose(torch.logsumexp(both, 0), lse, rtol=1e-5, atol=1e-5)
    assert torch.allclose(joined, whole.double(), rtol=2e-3, atol=2e-3)


@pytest.mark.parametrize("lengths,cache", [([300, 2000, 10], "same"), ([4000], "int8"), ([40] * 30, "float8_e4m3fn")])
def test_same_bits_every_time_and_in_a_graph(cuda, lengths, cache):
    case = _Case(cuda, lengths, 16, 4, 128, 16, "bfloat16", cache)
    first, lse = case.run()
    for _ in range(5):
        out, again = case.run()
        assert torch.equal(out, first) and torch.equal(lse, again)
    n = torch.tensor(lengths, dtype=torch.int32, device=cuda)
    table = case.table.to(cuda)
    kernel = tl.paged_attention_decode(len(lengths), 16, **case.sizes)
    out = kernel(case.q, *case.pool(), table, n)
    assert torch.equal(out, first)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = kernel(case.q, *case.pool(), table, n)
    for shorter in (0, 1, 7, 0):
        # lengths change between replays, as in a decode loop
        n.copy_(torch.tensor([max(0, x - shorter) for x in lengths], dtype=torch.int32))
        want = kernel(case.q, *case.pool(), table, n)
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_offsets_beyond_32_bits(cuda):
    """A cache of more than 2^32 elements: the pages at its end, read by the attention and the read, written by the write."""
    page_size, kv_heads, dim = 1024, 8, 256
    pages = 2**32 // (page_size * kv_heads * dim) + 2
    try:
        kc, vc = (torch.zeros((pages, kv_heads, page_size, dim), dtype=torch.int8, device=cuda) for _ in range(2))
    except torch.OutOfMemoryError:
        pytest.skip("not enough memory")
    ks, vs = (torch.zeros((pages, kv_heads, page_size), device=cuda) for _ in range(2))
    pool = dict(kv_heads=kv_heads, head_dim=dim, pages=pages, page_size=page_size, dtype="bfloat16", cache_dtype="int8")
    tokens = 40
    gen = torch.Generator().manual_seed(3)
    k, v = (torch.randn((tokens, kv_heads, dim), generator=gen).bfloat16().to(cuda) for _ in range(2))
    slots = torch.arange(tokens, dtype=torch.int32, device=cuda) + (pages - 1) * page_size
    tl.kv_cache_write(tokens, **pool)(k, v, slots, kc, vc, ks, vs)
    assert (ks[:-1] == 0).all()
    table = torch.full((1, 1), pages - 1, dtype=torch.int32, device=cuda)
    rk, rv = tl.kv_cache_read(1, tokens, max_pages=1, **pool)(kc, vc, ks, vs, table, torch.tensor([0, tokens], dtype=torch.int32, device=cuda))
    for got, want in ((rk, k), (rv, v)):
        most = want.float().abs().amax(dim=-1, keepdim=True)
        assert ((got.float() - want.float()).abs() <= most * (0.5 / 127 + 2.0**-8)).all()
    q = torch.randn((1, 16, dim), generator=gen).bfloat16().to(cuda)
    out = tl.paged_attention_decode(1, 16, max_pages=1, **pool)(q, kc, vc, ks, vs, table, torch.tensor([tokens], dtype=torch.int32, device=cuda))
    want, _, spread = attention(q[0], *(tokens_of(c[-1:], s[-1:], [0], tokens) for c, s in ((kc, ks), (vc, vs))), dim**-0.5)
    assert ((out[0].cpu().double() - want).abs() <= attention_bound(want, spread, out.dtype, torch.int8)).all()


def _ragged(n, longest, seed):
    gen = torch.Generator().manual_seed(seed)
    lengths = (torch.rand(n, generator=gen) ** 3 * longest).int().tolist()
    lengths[n // 2], lengths[n // 3] = longest, 0
    return lengths


@pytest.mark.parametrize("lengths,heads,kv_heads,dim,page_size,cache,window,sinks", [
    # more sequences than a workgroup has threads, several a thread; nothing that can be cut
    (_ragged(700, 120, 1), 2, 1, 64, 8, "same", 0, False),
    # ... and one among them that is
    (_ragged(530, 6000, 2), 2, 2, 64, 16, "int8", 0, True),
    # few columns cut into hundreds of pieces, more than a lane group takes at once
    ([70000, 3], 6, 2, 64, 128, "float8_e4m3fn", 0, True),
    ([33000], 3, 1, 128, 64, "same", 0, False),
    # many columns, some cut: the join of a group a head
    (_ragged(150, 3000, 3), 48, 16, 64, 16, "same", 0, True),
    # whole columns of several units, and of one more unit than that
    ([2048, 1, 2047, 700] * 4, 32, 32, 64, 64, "same", 0, False),
    ([2049, 1, 2048, 700] * 4, 32, 32, 64, 64, "same", 0, False),
    ([512, 513, 511] * 3, 4, 4, 80, 32, "float8_e4m3fn", 0, False),
    # two blocks of 16 heads, and three, and a wide head that takes them one by one
    ([900, 20], 71, 1, 64, 16, "same", 0, True),
    ([5000], 33, 1, 128, 16, "int8", 0, False),
    ([1300, 0, 77], 40, 1, 192, 16, "same", 0, False),
    # windows that are cut and windows that are not
    ([9000, 300, 40], 8, 2, 128, 16, "int8", 3001, True),
    ([9000, 300, 40], 8, 2, 128, 16, "same", 481, False),
], ids=lambda v: f"{len(v)}x{max(v)}" if isinstance(v, list) else str(v))
def test_shares(cuda, lengths, heads, kv_heads, dim, page_size, cache, window, sinks):
    """Batches whose work is cut in every way that there is."""
    print(f"shares n={len(lengths)} longest={max(lengths)} {heads}/{kv_heads}x{dim} page {page_size} {cache} window {window}", flush=True)
    case = _Case(cuda, lengths, heads, kv_heads, dim, page_size, "bfloat16", cache)
    case.check(window=window, sinks=sinks)
    first, _ = case.run(window, sinks)
    for _ in range(2):
        assert torch.equal(case.run(window, sinks)[0], first)
