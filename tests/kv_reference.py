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
    x = cache.float().cpu().double()
    if scale is not None:
        x = x * scale.cpu().double()[..., None]
    out = torch.full((length, cache.shape[1], cache.shape[3]), math.nan, dtype=torch.float64)
    for t in range(0, length, size):
        page, n = int(pages[t // size]), min(size, length - t)
        if 0 <= page < cache.shape[0]:
            out[t : t + n] = x[page, :, :n].transpose(0, 1)
    return out


def attention(q, keys, values, scale, window=0, sinks=None, there=None):
    """One sequence: q [heads, head_dim], keys and values [length, kv_heads, head_dim] in 64 bits, there [length] truth
    values.  Returns out, lse and sum_t p_t |v_t| / sum p, which rounded weights are off by in proportion."""
    heads, dim = q.shape
    length, kv_heads = keys.shape[:2]
    out, spread = torch.zeros((heads, dim), dtype=torch.float64), torch.zeros((heads, dim), dtype=torch.float64)
    lse = torch.full((heads,), -math.inf, dtype=torch.float64)
    first = max(0, length - window) if window else 0
    live = torch.arange(length) >= first
    if there is not None:
        live &= there
    for h in range(heads):
        k, v = keys[live][:, h * kv_heads // heads], values[live][:, h * kv_heads // heads]
        s = (k @ q[h].cpu().double()) * scale
        extra = s.new_tensor([float(sinks[h])]) if sinks is not None else s.new_empty(0)
        both = torch.cat([s, extra])
        if not len(both):
            continue
        lse[h] = torch.logsumexp(both, 0)
        p = torch.exp(s - lse[h])
        out[h], spread[h] = p @ v, p @ v.abs()
    return out, lse, spread


def attention_bound(out, spread, dtype, held):
    """|kernel - exact|: the output's rounding; a weight's rounding to the type of the products (fp16 where the cache is
    quantised) and the fp32 score, exponential and sums (2^-14 for scores to some ten); values below fp16's normal range,
    relative to the largest, only where quantised."""
    weights = HALF_ULP[dtype if held == dtype else torch.float16] + 2.0**-14
    return HALF_ULP[dtype] * out.abs() + weights * spread + 2.0**-20 * spread.amax().clamp(min=1e-30)
