"""Attention of one new token where its numbers are far apart: scores, value scales and weights over the whole range that fp32 holds."""

import math

import pytest
import torch

import tilelang_amd as tl
from kv_reference import attention, attention_bound, tokens_of

pytestmark = pytest.mark.gpu

DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float8_e4m3fn": torch.float8_e4m3fn, "int8": torch.int8}
#: heads, kv_heads, head_dim: heads that share lanes, one block of 16 and two of them
HEADS = [(4, 1, 64), (12, 1, 64), (6, 2, 128), (20, 1, 128), (5, 1, 256), (18, 1, 160)]


class _Sequence:
    """One sequence in pages in order: keys and values [length, kv_heads, head_dim] as numbers of the cache's type, scales
    [length] or None, queries [heads, head_dim]."""

    def __init__(self, cuda, q, keys, values, held, key_scale=None, value_scale=None, page_size=16):
        length, kv_heads, dim = keys.shape
        self.length, self.q, self.dim, self.held = length, q.to(cuda)[None], dim, held
        pages = -(-length // page_size)
        self.buffers = []
        for x, s in ((keys, key_scale), (values, value_scale)):
            whole = torch.zeros((pages * page_size, kv_heads, dim))
            whole[:length] = x.float()
            cache = whole.view(pages, page_size, kv_heads, dim).transpose(1, 2).contiguous().to(held).to(cuda)
            scale = None
            if s is not None:
                scale = torch.zeros((pages * page_size, kv_heads))
                scale[:length] = s[:, None]
                scale = scale.view(pages, page_size, kv_heads).transpose(1, 2).contiguous().to(cuda)
            self.buffers.append((cache, scale))
        self.table = torch.arange(pages, dtype=torch.int32, device=cuda)[None]
        name = {v: k for k, v in DTYPES.items()}
        self.sizes = dict(kv_heads=kv_heads, head_dim=dim, pages=pages, page_size=page_size, max_pages=pages, dtype=name[q.dtype],
                          cache_dtype=None if held == q.dtype else name[held])

    def run(self, scale, length=None, max_pages=None):
        (kc, ks), (vc, vs) = self.buffers
        n = torch.tensor([self.length if length is None else length], dtype=torch.int32, device=kc.device)
        table = self.table if max_pages is None else torch.nn.functional.pad(self.table, (0, max_pages - self.table.shape[1]), value=-1)
        sizes = self.sizes | dict(max_pages=table.shape[1])
        kernel = tl.paged_attention_decode(1, self.q.shape[1], scale=scale, with_lse=True, **sizes)
        out, lse = kernel(self.q, *((kc, vc) if ks is None else (kc, vc, ks, vs)), table, n)
        return out[0].cpu().double(), lse[0].cpu().double()

    def exact(self, scale):
        k, v = (tokens_of(c, s, self.table[0].cpu(), self.length) for c, s in self.buffers)
        return attention(self.q[0], k, v, scale)


def _coded(cuda, heads, kv_heads, dim, held, scores, value_scale, codes=None, dtype=torch.bfloat16):
    """A quantised sequence whose tokens' scores are `scores` for every head: queries of ones on codes of 16, scale 1 / (16 head_dim)."""
    n = len(scores)
    q = torch.ones((heads, dim), dtype=dtype)
    keys = torch.full((n, kv_heads, dim), 16.0)
    if codes is None:
        codes = torch.randint(-120, 121, (n, kv_heads, dim), generator=torch.Generator().manual_seed(n + dim)).float()
    return _Sequence(cuda, q, keys, codes, held, torch.tensor(scores), torch.tensor(value_scale)), 1 / (16 * dim)


@pytest.mark.parametrize("cache", ["float8_e4m3fn", "int8"])
@pytest.mark.parametrize("heads,kv_heads,dim", HEADS)
@pytest.mark.parametrize("length", [20, 300])
@pytest.mark.parametrize("best", ["first", "later"])
def test_best_token_without_a_value(cuda, best, length, heads, kv_heads, dim, cache):
    """The token that outweighs all others has a value scale of zero, as a head of zeros is stored: what the others leave is tiny, and a
    number.  First: among the first tokens, the others 86 below (times their scale out of fp32's normal range).  Later: 200 above those
    that came before."""
    print(f"best token {best} of {length}, {heads}/{kv_heads}x{dim} {cache}", flush=True)
    scores, scales = [0.0] * length, [2.0**-5] * length
    for t in (3,) if best == "first" else range(min(140, length - 5), length):
        scores[t], scales[t] = (86.0 if best == "first" else 200.0), 0.0
    case, scale = _coded(cuda, heads, kv_heads, dim, DTYPES[cache], scores, scales)
    out, lse = case.run(scale)
    want, want_lse, spread = case.exact(scale)
    assert torch.isfinite(out).all()
    assert ((out - want).abs() <= attention_bound(want, spread, torch.bfloat16, case.held)).all()
    assert ((lse - want_lse).abs() <= 2.0**-16 * (1 + want_lse.abs())).all()


@pytest.mark.parametrize("cache", ["float8_e4m3fn", "int8"])
@pytest.mark.parametrize("heads,kv_heads,dim", HEADS)
@pytest.mark.parametrize("sign", ["all", "some"])
def test_negative_value_scales(cuda, sign, heads, kv_heads, dim, cache):
    """value = code * scale, whatever the scale's sign and size."""
    print(f"negative scales ({sign}) {heads}/{kv_heads}x{dim} {cache}", flush=True)
    n, gen = 333, torch.Generator().manual_seed(dim)
    for exponent in (-40, 0, 30):
        scales = torch.exp2(exponent + 4 * torch.rand(n, generator=gen))
        scales = -scales if sign == "all" else scales * torch.where(torch.rand(n, generator=gen) < 0.3, -64.0, 1.0)
        case, scale = _coded(cuda, heads, kv_heads, dim, DTYPES[cache], torch.randn(n, generator=gen).tolist(), scales.tolist())
        out, _ = case.run(scale)
        want, _, spread = case.exact(scale)
        assert ((out - want).abs() <= attention_bound(want, spread, torch.bfloat16, case.held)).all(), exponent


def _one_and_many(cuda, heads, kv_heads, dim, dtype, cache, n, gap):
    """One early token of a value of zero, and n others whose scores lie `gap` to `gap` - 1 below its score."""
    gen = torch.Generator().manual_seed(n + dim)
    below = gap - torch.rand(n, generator=gen)
    values = 0.5 + torch.rand((n, kv_heads, dim), generator=gen)  # (of one sign, so that what is lost adds up)
    values[5] = 0.0
    if cache != "same":
        scores = gap - below
        scores[5] = gap
        return _coded(cuda, heads, kv_heads, dim, DTYPES[cache], scores.tolist(), [2.0**-6] * n, (values * 60).round(), DTYPES[dtype])
    keys = (gap - below)[:, None, None].expand(n, kv_heads, dim).clone()
    keys[5] = gap
    held = DTYPES[dtype]
    return _Sequence(cuda, torch.ones((heads, dim), dtype=held), keys.to(held), values.to(held), held), 1 / dim


@pytest.mark.parametrize("dtype,cache", [("float16", "same"), ("float16", "float8_e4m3fn"), ("bfloat16", "int8"), ("bfloat16", "same")])
@pytest.mark.parametrize("heads,kv_heads,dim", HEADS)
@pytest.mark.parametrize("gap", [12.0, 18.5])
def test_many_light_tokens_beside_a_heavy_one(cuda, gap, heads, kv_heads, dim, dtype, cache):
    """Weights of e^-18 and less of the largest, below what fp16 holds beside 1, whose values are all that there is."""
    print(f"light tokens {gap} below, {heads}/{kv_heads}x{dim} {dtype} {cache}", flush=True)
    case, scale = _one_and_many(cuda, heads, kv_heads, dim, dtype, cache, 3000, gap)
    out, _ = case.run(scale)
    want, _, spread = case.exact(scale)
    # the output's rounding (fp16's smallest steps among them), fp32 scores of up to 20 and sums: 2^-14
    half = 2.0**-11 if dtype == "float16" else 2.0**-8
    assert ((out - want).abs() <= half * want.abs() + 2.0**-25 + 2.0**-14 * spread).all(), ((out - want).abs() / spread).max()


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("cache", ["same", "float8_e4m3fn", "int8"])
@pytest.mark.parametrize("heads,kv_heads,dim", HEADS)
@pytest.mark.parametrize("length", [3, 17, 70])
def test_weights_keep_their_bits(cuda, length, heads, kv_heads, dim, cache, dtype):
    """The weights' rounding does not show beside the output's: 2^-16 of each where they go into the product in two parts of bf16 (less in
    fp16), and 2^-14 from fp32 scores, exponentials and sums."""
    print(f"weights' bits {length} {heads}/{kv_heads}x{dim} {dtype} {cache}", flush=True)
    held = DTYPES[dtype if cache == "same" else cache]
    gen = torch.Generator().manual_seed(length * dim)
    q = torch.randn((heads, dim), generator=gen).to(DTYPES[dtype])
    keys, values = torch.randn((2, length, kv_heads, dim), generator=gen)
    scales = (None, None)
    if cache != "same":
        keys, values, scales = (keys * 40).round(), (values * 40).round(), (torch.rand((2, length), generator=gen) + 0.5) / 40
    case = _Sequence(cuda, q, keys, values, held, *scales)
    out, _ = case.run(dim**-0.5)
    want, _, spread = case.exact(dim**-0.5)
    half = 2.0**-11 if dtype == "float16" else 2.0**-8
    assert ((out - want).abs() <= half * want.abs() + 2.0**-25 + (2.0**-14 + 2.0**-16) * spread).all(), ((out - want).abs() / spread).max()


@pytest.mark.parametrize("cache", ["float8_e4m3fn", "int8"])
@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 1, 128), (16, 1, 256), (4, 1, 64), (20, 2, 128)])
@pytest.mark.parametrize("mean,width", [(3.0, 2.0), (12.0, 8.0)])
def test_queries_that_are_not_centred(cuda, mean, width, heads, kv_heads, dim, cache):
    """Queries whose elements have a mean, keys with one channel far out: the score is a small part of what such queries would sum up to
    with every code moved by a constant."""
    print(f"queries around {mean} {heads}/{kv_heads}x{dim} {cache}", flush=True)
    gen, n = torch.Generator().manual_seed(dim + int(mean)), 200
    q = (mean + width * torch.randn((heads, dim), generator=gen)).to(torch.float16)
    keys, values = torch.randn((2, n, kv_heads, dim), generator=gen)
    keys[..., 7] = 30.0
    top = 127.0 if cache == "int8" else 448.0
    most = keys.abs().amax(dim=(1, 2))
    codes = keys * (top / most)[:, None, None]
    case = _Sequence(cuda, q, codes.round() if cache == "int8" else codes, (values * 30).round(), DTYPES[cache], most / top,
                     torch.full((n,), 1 / 30))
    out, lse = case.run(dim**-0.5)
    want, want_lse, spread = case.exact(dim**-0.5)
    assert ((lse - want_lse).abs() <= 2.0**-16 * (1 + want_lse.abs())).all(), (lse - want_lse).abs().max()
    # a score's error is a weight's, relative: as above, of scores of up to a hundred
    assert ((out - want).abs() <= 2.0**-11 * want.abs() + 2.0**-25 + 2.0**-13 * spread).all(), ((out - want).abs() / spread).max()


@pytest.mark.parametrize("cache", ["same", "int8"])
@pytest.mark.parametrize("length,max_pages", [(1, 1), (40, 3), (700, 60), (2000, 200)])
@pytest.mark.parametrize("what", ["query", "keys"])
def test_nothing_but_nan(cuda, what, length, max_pages, cache):
    """A head all of whose scores are NaN has no logarithm of a sum: NaN, not the -inf of a head that sees no token."""
    print(f"nan {what} {length} of {max_pages} pages {cache}", flush=True)
    heads, kv_heads, dim = 6, 2, 64
    gen = torch.Generator().manual_seed(length)
    q = torch.randn((heads, dim), generator=gen).half()
    keys, values = torch.randn((2, length, kv_heads, dim), generator=gen)
    scales = (None, None) if cache == "same" else (torch.full((length,), 1 / 40), torch.full((length,), 1 / 40))
    if what == "query":
        q[4] = math.nan
    elif cache == "same":
        keys[:, 1] = math.nan
    else:
        keys, values = (keys * 40).round(), (values * 40).round()
    case = _Sequence(cuda, q, keys, values, torch.float16 if cache == "same" else torch.int8, *scales)
    if what == "keys" and cache == "int8":
        case.buffers[0][1][:, 1] = math.nan
    out, lse = case.run(0.125, max_pages=max(max_pages, -(-length // 16)))
    lost = torch.zeros(heads, dtype=torch.bool)
    lost[4 if what == "query" else slice(3, 6)] = True
    assert torch.isnan(out[lost]).all() and torch.isnan(lse[lost]).all()
    assert torch.isfinite(out[~lost]).all() and torch.isfinite(lse[~lost]).all()
    out, lse = case.run(0.125, length=0, max_pages=max(max_pages, -(-length // 16)))
    assert (out == 0).all() and (lse == -math.inf).all()
