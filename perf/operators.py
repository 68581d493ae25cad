"""What the operators around a decode step's projections are measured on: rotary positions, the paged key-value cache as it
is written and read back, and the attention of one new token over it.

``listed()`` names twelve cases, ``draw(rng)`` gives more of the same ranges; ``prepare`` makes what a serving (or, for
the rotation's gradient, a training) program holds before the call, ``run`` is one pass through one operator: with
``own`` through the package's kernel objects, else in plain torch in 32 bits.  ``exact`` is the definition in 64 bits.

A sequence's cache pages are scattered over the pool, its table names more pages than it has tokens (-1 beyond them), and
what lies behind a sequence's last token in its last page is NaN, as a reused page may well hold.
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float8_e4m3fn": torch.float8_e4m3fn, "int8": torch.int8}
TOP = {"float8_e4m3fn": 448.0, "int8": 127.0}  # the largest magnitude of a code
SMALLEST = 2.0**-100  # a head whose largest magnitude is below is stored as zeros


def _rotary(name, tokens, heads, head_dim, rotary_dim, interleaved, dtype, gradient=False, more_heads=0):
    return {"name": name, "kind": "rotary", "tokens": tokens, "heads": heads, "head_dim": head_dim, "rotary_dim": rotary_dim,
            "interleaved": interleaved, "dtype": dtype, "gradient": gradient, "more_heads": more_heads}


def _cache(name, sequences, new, longest, heads, kv_heads, head_dim, rotary_dim, dtype, cache, back, ragged=True, page=16, interleaved=False):
    return {"name": name, "kind": "cache", "sequences": sequences, "new": new, "longest": longest, "ragged": ragged, "heads": heads,
            "kv_heads": kv_heads, "head_dim": head_dim, "rotary_dim": rotary_dim, "interleaved": interleaved, "dtype": dtype,
            "cache": cache, "back": back, "page": page}


def _attention(name, sequences, longest, heads, kv_heads, head_dim, dtype, cache, ragged=False, window=0, sinks=False, page=16):
    return {"name": name, "kind": "attention", "sequences": sequences, "longest": longest, "ragged": ragged, "heads": heads,
            "kv_heads": kv_heads, "head_dim": head_dim, "dtype": dtype, "cache": cache, "window": window, "sinks": sinks, "page": page}


def listed():
    return [
        # the queries and keys of one new token: the smallest call, latency counts
        _rotary("rotary one token", 1, 40, 128, 128, False, "bfloat16"),
        # queries and keys of a batch of prompts, rotated out of a fused q/k/v projection's rows (8 heads of values beside them)
        _rotary("rotary prompt", 4096, 40, 128, 128, False, "float16", more_heads=8),
        # a training step's gradient through the rotation: interleaved pairs, part of an 80-wide head, odd length
        _rotary("rotary gradient", 7999, 64, 80, 32, True, "bfloat16", gradient=True),
        # sixteen sequences decoding: each writes its one new token, rotated on the way, into a 16-bit cache
        _cache("cache one step", 16, 1, 500, 32, 8, 128, 128, "bfloat16", "bfloat16", False),
        # a chunk of four prompts goes into an fp8 cache, and their whole contexts come back for the chunk's own attention
        _cache("cache chunk fp8", 4, 512, 8192, 32, 8, 128, 128, "bfloat16", "float8_e4m3fn", True),
        # odd chunks of many short prompts, interleaved pairs on part of a 96-wide head, int8, larger pages
        _cache("cache chunk int8", 48, 37, 1100, 24, 12, 96, 48, "float16", "int8", True, page=64, interleaved=True),
        # one long context read back whole, nothing written (a prefix shared with a new request)
        _cache("cache long read", 1, 0, 131071, 32, 8, 128, 0, "bfloat16", "float8_e4m3fn", True),
        # one sequence with a short context: latency counts
        _attention("attention one sequence", 1, 1000, 32, 8, 128, "float16", "float16"),
        # one sequence with a long context: eight heads of keys and values for 256 compute units
        _attention("attention long context", 1, 131071, 64, 8, 128, "bfloat16", "bfloat16"),
        # a serving batch, lengths from none (an empty place of the batch) to 16 thousand, fp8
        _attention("attention ragged batch", 64, 16000, 32, 8, 128, "bfloat16", "float8_e4m3fn", ragged=True),
        # a layer with a sliding window and sinks, 64-wide heads
        _attention("attention window", 96, 4099, 64, 8, 64, "bfloat16", "bfloat16", ragged=True, window=128, sinks=True, page=64),
        # the largest batch: 128 sequences of 8192 tokens, int8
        _attention("attention large batch", 128, 8192, 32, 8, 128, "float16", "int8", page=32),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(lo * ((hi + 1) / lo) ** rng.random())))


def draw(rng):
    # widths that the package's own matrices have none of are left out
    while (case := _drawn(rng)) and 3 << 10 in _widths(case):
        pass
    return case


def _widths(case):
    return [v for v in case.values() if type(v) is int] + [case["head_dim"] * n for n in
            (case["heads"], case["heads"] + case.get("more_heads", 0), case.get("kv_heads", 0), case["heads"] + 2 * case.get("kv_heads", 0))]


def _drawn(rng):
    dtype = rng.choice(("float16", "bfloat16"))
    kind = rng.choice(("rotary", "cache", "attention"))
    head_dim = rng.choice((64, 80, 96, 128, 128, 128, 256))
    kv_heads = rng.choice((1, 2, 4, 8, 8, 12, 16))
    heads = kv_heads * rng.choice((1, 2, 3, 4, 7, 8))
    part = head_dim if rng.random() < 0.6 else rng.randrange(1, head_dim // 16) * 16
    interleaved = rng.random() < 0.4
    cache = rng.choice((dtype, "float8_e4m3fn", "int8"))
    page = rng.choice((8, 16, 16, 32, 64, 128))
    if kind == "rotary":
        heads += kv_heads
        tokens = _log(rng, 1, min(8192, 7999 * 64 * 80 // (heads * head_dim)))
        more = rng.choice((0, kv_heads))
        case = _rotary("", tokens, heads, head_dim, part, interleaved, dtype, rng.random() < 0.3, more)
    else:
        sequences = _log(rng, 1, 128)
        ragged = sequences > 1 and rng.random() < 0.7
        # nothing costs more than the largest listed case of its kind
        most = (131071 * 8 * 128 if kind == "cache" else 128 * 8192 * 8 * 128) // (kv_heads * head_dim * sequences)
        longest = _log(rng, 1, min(131071, most))
        if kind == "cache":
            new = rng.choice((0, 1, _log(rng, 1, 512), _log(rng, 1, 512)))
            if not new:
                back = True
            else:  # codes in 8 bits come back as values
                new, back = min(new, longest), cache != dtype or rng.random() < 0.5
            rotary_dim = 0 if not new or rng.random() < 0.2 else part
            while new and sequences * new * (heads + 2 * kv_heads) * head_dim > 131071 * 8 * 128:
                new = (new + 1) // 2
            case = _cache("", sequences, new, longest, heads, kv_heads, head_dim, rotary_dim, dtype, cache, back, ragged, page, interleaved)
        else:
            case = _attention("", sequences, longest, heads, kv_heads, head_dim, dtype, cache, ragged,
                              rng.choice((0, 0, 0, _log(rng, 16, 4096))), rng.random() < 0.3, page)
    del case["name"]
    return case


# ---- inputs --------------------------------------------------------------------------------------------------------------


def _lengths(case):
    """Tokens of each sequence, the longest first; ragged: down by squares, as a serving batch's are, and the last of
    sixteen or more none at all."""
    n, longest = case["sequences"], case["longest"]
    if not case["ragged"]:
        return [longest] * n
    least = case.get("new", 0)
    lengths = [max(least, int(longest * ((n - i) / n) ** 2), 1) for i in range(n)]
    if n >= 16 and not least:
        lengths[-1] = 0
    return lengths


class _Inputs:
    """Random inputs on the GPU, from the seed alone."""

    def __init__(self, seed):
        self.dev = torch.device("cuda")
        self.gen = torch.Generator(device=self.dev)
        self.gen.manual_seed(seed)

    def normal(self, *shape, dtype=torch.float32):
        return torch.randn(shape, dtype=torch.float32, device=self.dev, generator=self.gen).to(dtype)

    def order(self, n):
        return torch.randperm(n, device=self.dev, generator=self.gen)

    def ints(self, lo, hi, *shape):
        return torch.randint(lo, hi, shape, device=self.dev, generator=self.gen, dtype=torch.int32)

    def rotary_table(self, positions, rotary_dim, stretched):
        """cos | sin of position * 10000^(-2i/r); stretched: positions four times as close together, as a model that is
        run beyond the length that it was trained on has them."""
        i = torch.arange(rotary_dim // 2, dtype=torch.float64, device=self.dev)
        angle = torch.arange(positions, dtype=torch.float64, device=self.dev)[:, None] * 10000.0 ** (-2 * i / rotary_dim)
        if stretched:
            angle = angle / 4
        return torch.cat([angle.cos(), angle.sin()], dim=1).float()

    def cache(self, case, lengths):
        """Keys and values, their scales (or None), and the table of pages."""
        page, heads, dim, dtype = case["page"], case["kv_heads"], case["head_dim"], case["cache"]
        counts = [-(-n // page) for n in lengths]
        width = max(1, -(-case["longest"] * 3 // (2 * page)))
        pages = sum(counts) + 3
        count = torch.tensor(counts, device=self.dev)
        column = torch.arange(width, device=self.dev)[None]
        used = column < count[:, None]
        table = torch.full((len(lengths), width), -1, dtype=torch.int32, device=self.dev)
        table[used] = self.order(pages)[: sum(counts)].int()
        last = torch.tensor([max(0, n - 1) // page for n in lengths], device=self.dev)
        at = table[torch.arange(len(lengths), device=self.dev), last].long()
        length = torch.tensor(lengths, dtype=torch.int32, device=self.dev)
        stale = (torch.arange(page, device=self.dev)[None] >= (length - last * page)[:, None]) & (length > 0)[:, None]
        where = at[:, None].expand(-1, page)[stale], torch.arange(page, device=self.dev)[None].expand(len(lengths), -1)[stale]
        both, scales = [], []
        for _ in range(2):
            x = torch.empty((pages, heads, page, dim), dtype=DTYPES[dtype], device=self.dev)
            step = max(1, (1 << 26) // (heads * page * dim))
            for lo in range(0, pages, step):
                part = self.normal(min(step, pages - lo), heads, page, dim)
                if dtype == "int8":
                    part = (part * 40).round().clamp(-127, 127)
                elif dtype == "float8_e4m3fn":
                    part = (part * 120).clamp(-448, 448)
                x[lo : lo + step] = part.to(DTYPES[dtype])
            scale = None
            if dtype in TOP:
                scale = (0.5 + torch.rand((pages, heads, page), device=self.dev, generator=self.gen)) / (40 if dtype == "int8" else 120)
                scale[where[0], :, where[1]] = math.nan
            if dtype != "int8":  # a NaN in each type; int8's are in the scales
                raw = x.view(torch.uint8) if dtype == "float8_e4m3fn" else x.view(torch.int16)
                raw[where[0], :, where[1]] = 0x7F if dtype == "float8_e4m3fn" else -1
            both.append(x)
            scales.append(scale)
        return both[0], both[1], scales[0], scales[1], table


def prepare(case, seed):
    x = _Inputs(seed)
    state = {"case": dict(case)}
    dtype = DTYPES[case["dtype"]]
    if case["kind"] == "rotary":
        positions = 131072 if case["tokens"] > 512 else 8192
        wide = x.normal(case["tokens"], case["heads"] + case["more_heads"], case["head_dim"], dtype=dtype)
        state["x"] = wide[:, : case["heads"]]
        state["table"] = x.rotary_table(positions, case["rotary_dim"], case["tokens"] > 512)
        # prompts of a batch one behind the other, the first of them a continued one
        start = int(torch.randint(0, positions // 2, (1,), generator=x.gen, device=x.dev))
        state["positions"] = (torch.arange(case["tokens"], dtype=torch.int32, device=x.dev) + start) % (positions // 2 + 1)
        return state
    lengths = _lengths(case)
    state["keys"], state["values"], state["key_scale"], state["value_scale"], state["pages"] = x.cache(case, lengths)
    length = torch.tensor(lengths, dtype=torch.int32, device=x.dev)
    if case["kind"] == "attention":
        state["q"] = x.normal(len(lengths), case["heads"], case["head_dim"], dtype=dtype) * 2
        state["lengths"] = length
        state["sinks"] = x.normal(case["heads"]) if case["sinks"] else None
        return state
    state["starts"] = torch.cat([length.new_zeros(1), length.cumsum(0).int()])
    new, tokens = case["new"], case["new"] * len(lengths)
    if new:
        # the last `new` tokens of every sequence, one sequence behind the other
        position = ((length - new)[:, None] + torch.arange(new, device=x.dev)[None]).int()
        slots = state["pages"].gather(1, (position // case["page"]).long()) * case["page"] + position % case["page"]
        state["positions"], state["slots"] = position.reshape(-1).contiguous(), slots.reshape(-1).int().contiguous()
        wide = case["heads"] + 2 * case["kv_heads"] if case["rotary_dim"] else 2 * case["kv_heads"]
        state["qkv"] = x.normal(tokens, wide, case["head_dim"], dtype=dtype)
        if case["rotary_dim"]:
            state["table"] = x.rotary_table(case["longest"] + 1, case["rotary_dim"], False)
        else:
            both = state.pop("qkv")
            state["k"], state["v"] = both[:, : case["kv_heads"]].contiguous(), both[:, case["kv_heads"] :].contiguous()
    return state


# ---- the plain forms: torch in 32 bits -----------------------------------------------------------------------------------


def _rotate(x, table, positions, rotary_dim, interleaved, sign=1.0):
    """[tokens, heads, head_dim] in 32 bits, rotated."""
    half = rotary_dim // 2
    row = table[positions.long()][:, None]
    cos, sin = row[..., :half], row[..., half:] * sign
    turned, rest = x[..., :rotary_dim], x[..., rotary_dim:]
    a, b = (turned[..., 0::2], turned[..., 1::2]) if interleaved else (turned[..., :half], turned[..., half:])
    lo, hi = a * cos - b * sin, b * cos + a * sin
    both = torch.stack([lo, hi], dim=-1).flatten(-2) if interleaved else torch.cat([lo, hi], dim=-1)
    return torch.cat([both, rest], dim=-1)


def _write(cache, scales, x, slots, case):
    page, place = (slots // case["page"]).long(), (slots % case["page"]).long()
    name = case["cache"]
    if name not in TOP:
        cache[page, :, place] = x.to(cache.dtype)
        return
    most = x.abs().amax(dim=-1)
    factor = torch.where(most >= SMALLEST, TOP[name] / most, 0.0)
    code = x * factor[..., None]
    code = code.round().clamp(-127, 127).to(torch.int8) if name == "int8" else code.clamp(-448, 448).to(torch.float8_e4m3fn)
    cache.view(torch.uint8)[page, :, place] = code.view(torch.uint8)
    scales[page, :, place] = torch.where(most >= SMALLEST, most / TOP[name], 0.0)


def _values(cache, index, name):
    """The codes at an index, as numbers in 32 bits."""
    if name == "float8_e4m3fn":
        return cache.view(torch.uint8)[index].view(torch.float8_e4m3fn).float()
    return cache[index].float()


def _read(state, total):
    case, starts = state["case"], state["starts"]
    token = torch.arange(total, device=starts.device)
    sequence = torch.searchsorted(starts[1:].long(), token, right=True)
    position = token - starts[sequence]
    page, place = state["pages"][sequence, position // case["page"]].long(), position % case["page"]

    def rows(cache, scale):
        x = _values(cache, (page, slice(None), place), case["cache"])
        return (x if scale is None else x * scale[page, :, place][..., None]).to(DTYPES[case["dtype"]])

    return torch.stack([rows(state["keys"], state["key_scale"]), rows(state["values"], state["value_scale"])])


def _plain_cache(state):
    case, q = state["case"], None
    kv = case["kv_heads"]
    if case["new"]:
        if case["rotary_dim"]:
            x, q_heads = state["qkv"].float(), case["heads"]
            turned = _rotate(x[:, : q_heads + kv], state["table"], state["positions"], case["rotary_dim"], case["interleaved"])
            q, k, v = turned[:, :q_heads].to(DTYPES[case["dtype"]]), turned[:, q_heads:], x[:, q_heads + kv :]
        else:
            k, v = state["k"].float(), state["v"].float()
        _write(state["keys"], state["key_scale"], k, state["slots"], case)
        _write(state["values"], state["value_scale"], v, state["slots"], case)
    return q


def _plain_attention(state):
    case = state["case"]
    n, kv, dim, page = case["sequences"], case["kv_heads"], case["head_dim"], case["page"]
    pages = state["pages"][:, : -(-case["longest"] // page)].long().clamp(min=0)
    token = torch.arange(pages.shape[1] * page, device=pages.device)[None]
    length = state["lengths"][:, None]
    live = token < length
    if case["window"]:
        live = live & (token >= length - case["window"])

    def whole(cache, scale):  # [sequences, kv_heads, tokens, head_dim], zeros where no token lives
        x = _values(cache, pages, case["cache"])
        if scale is not None:
            x = x * scale[pages][..., None]
        return x.transpose(1, 2).reshape(n, kv, -1, dim).masked_fill_(~live[:, None, :, None], 0.0)

    q = state["q"].float().reshape(n, kv, -1, dim)
    scores = torch.matmul(whole(state["keys"], state["key_scale"]), q.transpose(2, 3).contiguous()).transpose(2, 3).contiguous()
    scores = (scores / math.sqrt(dim)).masked_fill_(~live[:, None, None], -math.inf)
    most = scores.amax(dim=-1, keepdim=True)
    sink = None if state["sinks"] is None else state["sinks"].reshape(1, kv, -1, 1)
    if sink is not None:
        most = torch.maximum(most, sink)
    most = torch.where(most == -math.inf, 0.0, most)
    p = torch.exp(scores - most)
    total = p.sum(dim=-1, keepdim=True)
    if sink is not None:
        total = total + torch.exp(sink - most)
    out = torch.matmul(p, whole(state["values"], state["value_scale"])) / torch.where(total == 0, 1.0, total)
    return out.reshape(n, -1, dim).to(DTYPES[case["dtype"]])


# ---- the package's kernel objects ----------------------------------------------------------------------------------------


def _kernels(state):
    """The kernel objects of a case, which a program makes once and keeps."""
    import tilelang_amd as tl

    case = state["case"]
    dim = case["head_dim"]
    if case["kind"] == "rotary":
        return (tl.rotary(case["tokens"], case["heads"], dim, positions=state["table"].shape[0], rotary_dim=case["rotary_dim"],
                          interleaved=case["interleaved"], inverse=case["gradient"], dtype=case["dtype"],
                          row_stride=(case["heads"] + case["more_heads"]) * dim),)
    pool = dict(kv_heads=case["kv_heads"], head_dim=dim, pages=state["keys"].shape[0], page_size=case["page"], dtype=case["dtype"],
                cache_dtype=case["cache"])
    width = state["pages"].shape[1]
    if case["kind"] == "attention":
        return (tl.paged_attention_decode(case["sequences"], case["heads"], max_pages=width, window=case["window"], sinks=case["sinks"], **pool),)
    write = back = None
    if case["new"] and case["rotary_dim"]:
        write = tl.rotary_kv_cache_write(case["sequences"] * case["new"], case["heads"], positions=state["table"].shape[0],
                                         rotary_dim=case["rotary_dim"], interleaved=case["interleaved"], **pool)
    elif case["new"]:
        write = tl.kv_cache_write(case["sequences"] * case["new"], **pool)
    if case["back"]:
        back = tl.kv_cache_read(case["sequences"], sum(_lengths(case)), max_pages=width, **pool)
    return write, back


def _own(state):
    case = state["case"]
    kernels = state.get("kernels")
    if kernels is None:
        kernels = state["kernels"] = _kernels(state)
    if case["kind"] == "rotary":
        return kernels[0](state["x"], state["table"], state["positions"])
    pool = (state["keys"], state["values"])
    if state["key_scale"] is not None:
        pool += (state["key_scale"], state["value_scale"])
    if case["kind"] == "attention":
        return kernels[0](state["q"], *pool, state["pages"], state["lengths"], *(() if state["sinks"] is None else (state["sinks"],)))
    q = None
    write, back = kernels
    if write is not None:
        if case["rotary_dim"]:
            q = write(state["qkv"], state["table"], state["positions"], state["slots"], *pool)
        else:
            write(state["k"], state["v"], state["slots"], *pool)
    return _cache_outputs(state, q, back(*pool, state["pages"], state["starts"]) if back is not None else None)


def _cache_outputs(state, q, kv):
    """The rotated queries, and the cache as it reads now: its tokens' values, or a 16-bit cache as it stands."""
    out = {} if q is None else {"q": q}
    return out | ({"kv": kv} if kv is not None else {"keys": state["keys"], "values": state["values"]})


def run(state):
    if own:
        return _own(state)
    case = state["case"]
    if case["kind"] == "rotary":
        return _rotate(state["x"].float(), state["table"], state["positions"], case["rotary_dim"], case["interleaved"],
                       -1.0 if case["gradient"] else 1.0).to(state["x"].dtype)
    if case["kind"] == "attention":
        return _plain_attention(state)
    q = _plain_cache(state)
    return _cache_outputs(state, q, _read(state, sum(_lengths(case))) if case["back"] else None)


# ---- what a pass cannot do without ---------------------------------------------------------------------------------------


def work(case):
    wide, dim = 2, case["head_dim"]
    if case["kind"] == "rotary":
        values = case["tokens"] * case["heads"] * dim
        return {"bytes": values * 2 * wide + case["tokens"] * (case["rotary_dim"] * 4 + 4),
                "flops": 3 * case["tokens"] * case["heads"] * case["rotary_dim"]}
    lengths = _lengths(case)
    # bytes of one token's keys and values as the cache holds them, with their scales
    held = 2 * case["kv_heads"] * (dim + 4 if case["cache"] in TOP else dim * wide)
    if case["kind"] == "attention":
        live = sum(min(n, case["window"]) if case["window"] else n for n in lengths)
        return {"bytes": live * held + 2 * case["sequences"] * case["heads"] * dim * wide, "flops": 4 * live * case["heads"] * dim}
    tokens = case["sequences"] * case["new"]
    heads = case["heads"] if case["rotary_dim"] else 0
    moved = tokens * ((2 * heads + 2 * case["kv_heads"]) * dim * wide + held + case["rotary_dim"] * 4 + 8)
    if case["back"]:
        moved += sum(lengths) * (held + 2 * case["kv_heads"] * dim * wide)
    return {"bytes": moved, "flops": 3 * tokens * (heads + 2 * case["kv_heads"]) * dim}


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------------


def _turned(x, table, positions, rotary_dim, interleaved, sign):
    """The rotation as products of complex numbers."""
    half = rotary_dim // 2
    x, row = x.double(), table[positions.long()].double()[:, None, :]
    turn = torch.complex(row[..., :half], sign * row[..., half:])
    pairs = torch.view_as_complex(x[..., :rotary_dim].reshape(*x.shape[:-1], half, 2)) if interleaved else torch.complex(x[..., :half].contiguous(), x[..., half:rotary_dim].contiguous())
    y = torch.view_as_real(pairs * turn)
    x = x.clone()
    x[..., :rotary_dim] = y.flatten(-2) if interleaved else torch.cat([y[..., 0], y[..., 1]], dim=-1)
    return x


def _tokens_of(state, b, length):
    """A sequence's keys and values in 64 bits, [tokens, kv_heads, head_dim]."""
    page = state["case"]["page"]
    pages = state["pages"][b, : -(-length // page)].tolist()

    def rows(cache, scale):
        x = cache.view(torch.uint8)[pages].view(cache.dtype).double() if cache.dtype == torch.float8_e4m3fn else cache[pages].double()
        if scale is not None:
            x = x * scale[pages].double()[..., None]
        return x.permute(0, 2, 1, 3).flatten(0, 1)[:length]

    return [rows(state["keys"], state["key_scale"]), rows(state["values"], state["value_scale"])]


def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "rotary":
        return _turned(state["x"], state["table"], state["positions"], case["rotary_dim"], case["interleaved"], -1.0 if case["gradient"] else 1.0)
    lengths = _lengths(case)
    dim, kv = case["head_dim"], case["kv_heads"]
    if case["kind"] == "attention":
        out = torch.zeros((len(lengths), case["heads"], dim), dtype=torch.float64, device="cuda")
        for b, n in enumerate(lengths):
            if not n:
                continue
            k, v = (t[-case["window"] :] if case["window"] else t for t in _tokens_of(state, b, n))
            q = state["q"][b].double().reshape(kv, -1, dim)
            scores = (q @ k.permute(1, 2, 0).contiguous()) / math.sqrt(dim)
            if state["sinks"] is not None:  # one more score, whose value is nothing
                scores = torch.cat([scores, state["sinks"].double().reshape(kv, -1, 1)], dim=2)
            p = torch.softmax(scores, dim=2)[..., : k.shape[0]]
            out[b] = (p @ v.transpose(0, 1).contiguous()).reshape(-1, dim)
        return out
    q, top = None, TOP.get(case["cache"])
    new = []
    if case["new"]:
        if case["rotary_dim"]:
            x = state["qkv"]
            turned = _turned(x[:, : case["heads"] + kv], state["table"], state["positions"], case["rotary_dim"], case["interleaved"], 1.0)
            q, k, v = turned[:, : case["heads"]], turned[:, case["heads"] :], x[:, case["heads"] + kv :].double()
        else:
            k, v = state["k"].double(), state["v"].double()
        for x in (k, v):
            if top:  # what the codes stand for
                scale = x.abs().amax(dim=-1, keepdim=True) / top
                code = x / scale
                x = (code.round() if case["cache"] == "int8" else code.float().to(torch.float8_e4m3fn).double()) * scale
            new.append(x)
    if not case["back"]:
        out = {"q": q} if q is not None else {}
        for name, x in zip(("keys", "values"), new):
            # a 16-bit cache in 64 bits, its new tokens' places as they would be without rounding
            whole = state[name].double()
            for t, slot in enumerate(state["slots"].tolist()):
                whole[slot // case["page"], :, slot % case["page"]] = x[t]
            out[name] = whole
        return out
    rows = [[], []]
    for b, n in enumerate(lengths):
        for k, x in enumerate(_tokens_of(state, b, n)):
            if case["new"]:
                x[n - case["new"] :] = new[k][b * case["new"] : (b + 1) * case["new"]]
            rows[k].append(x)
    kv = torch.stack([torch.cat(r) for r in rows])
    return {"kv": kv} if q is None else {"q": q, "kv": kv}
