"""Plain 64-bit forms of the rotation, the paged cache and the attention over it, and the bounds of their kernels' errors."""

import math

import torch

#: half a unit in the last place, relative
HALF_ULP = {torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}
TOP = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}


def rotate(x, table, positions, rotary_dim, interleaved, inverse=False):
    """x [tokens, heads, head_dim] turned, in 64 bits, and the bound of an fp32 product and sum's error."""
    x, row = x.double(), table.double()[positions.long()][:, None]
    half = rotary_dim // 2
    c, s = row[..., :half], row[..., half:] * (-1.0 if inverse else 1.0)
    first = torch.arange(half, device=x.device) * (2 if interleaved else 1)
    second = first + (1 if interleaved else half)
    y, slack = x.clone(), torch.zeros_like(x)
    a, b = x[..., first], x[..., second]
    y[..., first], y[..., second] = a * c - b * s, b * c + a * s
    # a product, a fused product and sum: two roundings of at most |ac| + |bs|
    slack[..., first] = 2.0**-23 * ((a * c).abs() + (b * s).abs())
    slack[..., second] = 2.0**-23 * ((b * c).abs() + (a * s).abs())
    return y, slack


def fill_cache(gen, pages, kv_heads, page_size, head_dim, held, device):
    """Random keys or values [pages, kv_heads, page_size, head_dim] as the cache holds them, and scales or None."""
    x = torch.randn((pages, kv_heads, page_size, head_dim), generator=gen)
    if held == torch.int8:
        codes = (x * 40).round().clamp(-127, 127).to(torch.int8)
    elif held == torch.float8_e4m3fn:
        codes = (x * 100).clamp(-448, 448).to(held)
    else:
        return x.to(held).to(device), None
    return codes.to(device), ((0.5 + torch.rand((pages, kv_heads, page_size), generator=gen)) / 64).to(device)


def stale(cache, scale, page, place):
    """NaN into a page from a place on: what a reused page may hold."""
    if cache.dtype == torch.int8:
        cache[page, :, place:] = 77
    elif cache.dtype == torch.float8_e4m3fn:
        cache.view(torch.uint8)[page, :, place:] = 0x7F
    else:
        cache[page, :, place:] = math.nan
    if scale is not None:
        scale[page, :, place:] = math.nan


def tokens_of(cache, scale, pages, length):
    """The first tokens of a sequence in 64 bits, [length, kv_heads, head_dim]; pages that are not there: NaN."""
    size = cache.shape[2]
    ids = torch.as_tensor(pages)[: -(-length // size)].long().cpu()
    there = (ids >= 0) & (ids < cache.shape[0])
    at = ids.clamp(0, cache.shape[0] - 1).to(cache.device)
    raw = cache.view(torch.uint8 if cache.dtype.itemsize == 1 else torch.int16)
    x = raw[at].view(cache.dtype).float().cpu().double()
    if scale is not None:
        x = x * scale[at].cpu().double()[..., None]
    x[~there] = math.nan
    return x.transpose(1, 2).reshape(-1, cache.shape[1], cache.shape[3])[:length]


def attention(q, keys, values, scale, window=0, sinks=None, there=None):
    """One sequence: q [heads, head_dim], keys and values [length, kv_heads, head_dim] in 64 bits, there [length] truth
    values.  Returns out, lse and sum_t p_t |v_t| / sum p, which rounded weights are off by in proportion."""
    heads, dim = q.shape
    length, kv_heads = keys.shape[:2]
    live = torch.arange(length) >= (max(0, length - window) if window else 0)
    if there is not None:
        live &= there
    out, spread = torch.zeros((heads, dim), dtype=torch.float64), torch.zeros((heads, dim), dtype=torch.float64)
    lse = torch.full((heads,), -math.inf, dtype=torch.float64)
    group = heads // kv_heads
    for j in range(kv_heads):
        k, v, own = keys[live, j], values[live, j], slice(j * group, (j + 1) * group)
        scores = (q[own].cpu().double() @ k.T) * scale
        both = scores if sinks is None else torch.cat([scores, sinks[own].double()[:, None]], dim=1)
        if not both.shape[1]:
            continue
        lse[own] = torch.logsumexp(both, 1)
        p = torch.exp(scores - lse[own, None])
        out[own], spread[own] = p @ v, p @ v.abs()
    return out, lse, spread


def attention_bound(out, spread, dtype, held):
    """|kernel - exact|: the output's rounding; a weight's rounding to the type of the products (fp16 where the cache is
    quantised) and the fp32 score, exponential and sums (2^-14 for scores to some ten); values below fp16's normal range,
    relative to the largest, only where quantised."""
    weights = HALF_ULP[dtype if held == dtype else torch.float16] + 2.0**-14
    return HALF_ULP[dtype] * out.abs() + weights * spread + 2.0**-20 * spread.amax().clamp(min=1e-30)
