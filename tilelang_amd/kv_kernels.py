"""Kernel factories around a decode step's projections: rotary positions, the paged key-value cache as it is written and
read back, and the attention of one new token over it.

As in :mod:`kernels`, a factory takes sizes and types and returns a :class:`~tilelang_amd.adapter.KernelAdapter` bound to an
entry point of ``libdqgemm.so`` (``include/dqgemm.h``); its call checks every operand and launches on torch's current
stream.  The cache is two tensors ``[pages, kv_heads, page_size, head_dim]`` that the caller keeps (:class:`PagedKVCache`
does), in the activations' type or in 8 bits with fp32 scales ``[pages, kv_heads, page_size]``.
"""

from __future__ import annotations

import functools
import math

import torch

from . import _lib
from .adapter import KernelAdapter, KernelParam
from .kernels import _dtype

DT_F16, DT_BF16 = 0, 1
CACHE_F16, CACHE_BF16, CACHE_FP8, CACHE_I8 = range(4)

#: head sizes that the attention is built for
ATTENTION_HEAD_DIMS = (64, 80, 96, 112, 128, 160, 192, 256)


def _type16(fn: str, dtype) -> torch.dtype:
    d = _dtype(dtype)
    if d not in (torch.float16, torch.bfloat16):
        raise ValueError(f"{fn}: dtype must be float16 or bfloat16 (got {dtype!r})")
    return d


def _cache_type(fn: str, cache_dtype, dtype: torch.dtype) -> torch.dtype:
    if cache_dtype is None:
        return dtype
    d = torch.float8_e4m3fn if cache_dtype in ("float8_e4m3fn", torch.float8_e4m3fn) else _dtype(cache_dtype)
    if d not in (dtype, torch.float8_e4m3fn, torch.int8):
        raise ValueError(f"{fn}: cache_dtype must be dtype itself, float8_e4m3fn or int8 (got {cache_dtype!r} with {dtype})")
    return d


_FORMATS = {torch.float16: CACHE_F16, torch.bfloat16: CACHE_BF16, torch.float8_e4m3fn: CACHE_FP8, torch.int8: CACHE_I8}


def _positive(fn: str, **sizes) -> None:
    for name, value in sizes.items():
        if value <= 0:
            raise ValueError(f"{fn}: {name} must be positive (got {value})")


#: heads of all tokens that a call of the rotation, the write and the read takes
MAX_HEADS = 2**25


def _heads(fn: str, tokens: int, heads: int) -> None:
    if tokens * heads > MAX_HEADS and max(tokens, heads) < 2**31:  # (beyond: no size at all, see _kernel)
        raise ValueError(f"{fn}: {tokens} tokens of {heads} heads: at most {MAX_HEADS} heads in a call")


@functools.lru_cache(maxsize=64)
def attention_sequences(heads: int, kv_heads: int, tokens: int) -> int:
    """How many sequences a call of :func:`paged_attention_decode` takes whose page tables have room for ``tokens`` tokens: the library
    counts its work, a unit 128 tokens of a key-value head and 16 query heads and three more, in 31 bits, and such columns in 23."""
    columns = kv_heads * -(-(heads // kv_heads) // 16)
    return min(65535, (2**23 - 1) // columns, (2**31 - 2) // (columns * (tokens // 128 + 3)))


def _rotation(fn: str, head_dim: int, rotary_dim: int | None, positions: int) -> int:
    rotary_dim = head_dim if rotary_dim is None else rotary_dim
    if rotary_dim < 2 or rotary_dim % 2 or rotary_dim > head_dim:
        raise ValueError(f"{fn}: rotary_dim={rotary_dim} must be even and from 2 to head_dim={head_dim}")
    _positive(fn, positions=positions)
    return rotary_dim


class _Pool:
    """The cache's parameters and what the entry points are told about it."""

    def __init__(self, fn, kv_heads, head_dim, pages, page_size, dtype, cache_dtype):
        _positive(fn, kv_heads=kv_heads, pages=pages)
        if head_dim <= 0 or head_dim % 8 or head_dim > 256:
            raise ValueError(f"{fn}: head_dim={head_dim} must be a multiple of 8, at most 256")
        if not 8 <= page_size <= 1024 or page_size & (page_size - 1):
            raise ValueError(f"{fn}: page_size={page_size} must be a power of two from 8 to 1024")
        if pages * page_size >= 2**31:
            raise ValueError(f"{fn}: {pages} pages of {page_size} tokens: slots are 32-bit")
        self.dtype = _type16(fn, dtype)
        self.held = _cache_type(fn, cache_dtype, self.dtype)
        shape = (pages, kv_heads, page_size, head_dim)
        self.params = [KernelParam("KCache", self.held, shape), KernelParam("VCache", self.held, shape)]
        self.scaled = self.held.itemsize == 1
        if self.scaled:
            self.params += [KernelParam("KScale", torch.float32, shape[:3]), KernelParam("VScale", torch.float32, shape[:3])]
        self.ints = (DT_BF16 if self.dtype == torch.bfloat16 else DT_F16, _FORMATS[self.held])

    def slots(self, first: int) -> tuple:
        """The four pointer arguments of the cache, whose parameters begin at ``first``."""
        return (first, first + 1, first + 2, first + 3) if self.scaled else (first, first + 1, None, None)


def _kernel(name: str, entry: str, params: list, result_idx: list, slots: tuple, ints: tuple, f: float | None = None,
            workspace_bytes: int | None = None, workspace_idx=()) -> KernelAdapter:
    """The kernel object of an entry point whose arguments are ``slots`` (a parameter each; None: NULL), the workspace's
    bytes where it takes one, ``ints``, a float where it takes one, and the stream."""
    if not all(-(2**31) <= i < 2**31 for i in ints):  # (ctypes would keep the lower 32 bits)
        raise ValueError(f"{name}: sizes are 32-bit (got {max(ints, key=abs)})")

    def launch(ptrs, stream):
        middle = () if workspace_bytes is None else (workspace_bytes,)
        end = () if f is None else (f,)
        return getattr(_lib.get_library(), entry)(*(None if s is None else ptrs[s] for s in slots), *middle, *ints, *end, stream)

    return KernelAdapter(name, params, result_idx, launch, _lib.last_error, workspace_idx=workspace_idx,
                         native=(entry, slots, ints, f or 0.0, workspace_bytes or 0))


def rotary_table(positions: int, rotary_dim: int, base: float = 10000.0, scaling: str | None = None, factor: float = 1.0,
                 original_positions: int | None = None, low: float = 1.0, high: float = 4.0, device=None) -> torch.Tensor:
    """The table that :func:`rotary` and :func:`rotary_kv_cache_write` read: fp32 ``[positions, rotary_dim]``, for every
    position the cosines of its ``rotary_dim / 2`` angles ``position * f_i``, then their sines; angles in 64 bits.

    ``f_i = base ** (-2 i / rotary_dim)``.  ``scaling`` stretches it to ``factor`` times ``original_positions``, the length
    that a model was trained on:

    * ``"linear"``: ``f_i / factor`` (positions closer together);
    * ``"base"``: the base grows, ``base * factor ** (r / (r - 2))``: the slowest angle is slowed by ``factor``, the fastest not;
    * ``"bands"``: an angle that turns fewer than ``low`` times in ``original_positions`` is slowed by ``factor``, one that
      turns more than ``high`` times is kept, between them the share of each goes linearly with the turns;
    * ``"ramp"``: as ``"bands"``, but the share goes linearly with the index ``i`` between the (rounded out) indices whose
      angles turn ``high`` and ``low`` times, and cosines and sines are multiplied by ``0.1 ln(factor) + 1``, which
      sharpens the attention of a longer context.  Models that were trained with it mostly have ``high=32``: give their own.
    """
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError(f"rotary_table: rotary_dim={rotary_dim} must be even and at least 2")
    _positive("rotary_table", positions=positions, base=base, factor=factor)
    i = torch.arange(rotary_dim // 2, dtype=torch.float64, device=device)
    if scaling == "base":
        if rotary_dim == 2:
            raise ValueError("rotary_table: scaling 'base' needs rotary_dim of at least 4")
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    f = base ** (-2 * i / rotary_dim)
    magnitude = 1.0
    if scaling == "linear":
        f = f / factor
    elif scaling in ("bands", "ramp"):
        if not original_positions or original_positions <= 0 or not 0 < low < high:
            raise ValueError(f"rotary_table: scaling {scaling!r} needs original_positions and 0 < low < high")
        if scaling == "bands":
            kept = (original_positions * f / (2 * math.pi) - low) / (high - low)
        else:
            def index(turns):  # whose angle turns that often
                return rotary_dim * math.log(original_positions / (turns * 2 * math.pi)) / (2 * math.log(base))

            first, last = max(math.floor(index(high)), 0), min(math.ceil(index(low)), rotary_dim - 1)
            kept = 1 - (i - first) / max(last - first, 0.001)
            magnitude = 0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0
        kept = kept.clamp(0, 1)
        f = f * kept + f / factor * (1 - kept)
    elif scaling not in (None, "base"):
        raise ValueError(f"rotary_table: unknown scaling {scaling!r}")
    angle = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * f
    return (torch.cat([angle.cos(), angle.sin()], dim=1) * magnitude).float()


def rotary(tokens: int, heads: int, head_dim: int, positions: int, rotary_dim: int | None = None, interleaved: bool = False,
           inverse: bool = False, dtype="float16", row_stride: int | None = None, in_place: bool = False) -> KernelAdapter:
    """Rotary positions: ``out = kernel(x, Table, Positions)``, ``x`` and ``out`` ``[tokens, heads, head_dim]``, ``Table`` fp32
    ``[positions, rotary_dim]`` (:func:`rotary_table`), ``Positions`` int32 ``[tokens]``.

    The first ``rotary_dim`` elements of every head turn (all by default), the others are copied: element ``i`` with
    ``i + rotary_dim / 2``, or ``2 i`` with ``2 i + 1`` (``interleaved``).  ``inverse`` turns back, which is the gradient:
    ``dx = rotary(..., inverse=True)(dout, Table, Positions)``.  ``row_stride``: elements from one token's heads to the
    next one's where ``x`` is a view of wider rows (the queries and keys of a fused projection).  ``in_place``: ``x`` itself
    is turned and nothing returned.  A position outside of the table gives NaN.
    """
    fn = "rotary"
    _positive(fn, tokens=tokens, heads=heads)
    _heads(fn, tokens, heads)
    if head_dim <= 0 or head_dim % 8 or head_dim > 512:
        raise ValueError(f"{fn}: head_dim={head_dim} must be a multiple of 8, at most 512")
    rotary_dim = _rotation(fn, head_dim, rotary_dim, positions)
    t = _type16(fn, dtype)
    stride = heads * head_dim if row_stride is None else row_stride
    if stride < heads * head_dim or stride % 8:
        raise ValueError(f"{fn}: row_stride={stride} must be a multiple of 8 and at least {heads * head_dim}")
    x = KernelParam("x", t, (tokens, heads, head_dim), strides=None if stride == heads * head_dim else (stride, head_dim, 1))
    params = [x, KernelParam("Table", torch.float32, (positions, rotary_dim)), KernelParam("Positions", torch.int32, (tokens,))]
    if not in_place:
        params.append(KernelParam("out", t, (tokens, heads, head_dim)))
    ints = (tokens, heads, head_dim, rotary_dim, positions, stride, int(interleaved), int(inverse), DT_BF16 if t == torch.bfloat16 else DT_F16)
    return _kernel(fn, "call_rotary", params, [] if in_place else [3], (0, 1, 2, 0 if in_place else 3), ints)


def kv_cache_write(tokens: int, kv_heads: int, head_dim: int, pages: int, page_size: int, dtype="float16", cache_dtype=None) -> KernelAdapter:
    """New keys and values into the cache: ``kernel(k, v, Slots, KCache, VCache[, KScale, VScale])``, ``k`` and ``v``
    ``[tokens, kv_heads, head_dim]``, ``Slots`` int32 ``[tokens]`` = page * page_size + place (one that is negative or beyond
    the cache is not written).  A call's slots have to be distinct: a place that two tokens name holds parts of both.

    ``cache_dtype``: ``dtype`` itself (default), or ``"float8_e4m3fn"`` / ``"int8"`` with one fp32 scale a token and head:
    ``scale = max|x| / top``, ``code = round(x * (top / max|x|))``, top 448 / 127.  A head with an infinity or a NaN reads back
    as NaN.
    """
    fn = "kv_cache_write"
    _positive(fn, tokens=tokens)
    pool = _Pool(fn, kv_heads, head_dim, pages, page_size, dtype, cache_dtype)
    _heads(fn, tokens, 2 * kv_heads)
    shape = (tokens, kv_heads, head_dim)
    params = [KernelParam("k", pool.dtype, shape), KernelParam("v", pool.dtype, shape), KernelParam("Slots", torch.int32, (tokens,)), *pool.params]
    return _kernel(fn, "call_kv_cache_write", params, [], (0, 1, 2, *pool.slots(3)), (tokens, kv_heads, head_dim, pages, page_size, *pool.ints))


def rotary_kv_cache_write(tokens: int, heads: int, kv_heads: int, head_dim: int, pages: int, page_size: int, positions: int,
                          rotary_dim: int | None = None, interleaved: bool = False, dtype="float16", cache_dtype=None) -> KernelAdapter:
    """:func:`rotary` and :func:`kv_cache_write` in one launch on the rows of a fused projection:
    ``q = kernel(qkv, Table, Positions, Slots, KCache, VCache[, KScale, VScale])``, ``qkv`` ``[tokens, heads + 2 * kv_heads,
    head_dim]`` (queries, keys, values), ``q`` ``[tokens, heads, head_dim]`` the rotated queries; the rotated keys, quantised
    from fp32, and the values go into the cache, at slots that are distinct.
    """
    fn = "rotary_kv_cache_write"
    _positive(fn, tokens=tokens, heads=heads)
    pool = _Pool(fn, kv_heads, head_dim, pages, page_size, dtype, cache_dtype)
    _heads(fn, tokens, heads + 2 * kv_heads)
    rotary_dim = _rotation(fn, head_dim, rotary_dim, positions)
    params = [KernelParam("qkv", pool.dtype, (tokens, heads + 2 * kv_heads, head_dim)),
              KernelParam("Table", torch.float32, (positions, rotary_dim)), KernelParam("Positions", torch.int32, (tokens,)),
              KernelParam("Slots", torch.int32, (tokens,)), *pool.params, KernelParam("q", pool.dtype, (tokens, heads, head_dim))]
    q = len(params) - 1
    return _kernel(fn, "call_rotary_kv_cache_write", params, [q], (0, 1, 2, 3, q, *pool.slots(4)),
                   (tokens, heads, kv_heads, head_dim, rotary_dim, positions, pages, page_size, int(interleaved), *pool.ints))


def kv_cache_read(sequences: int, tokens: int, kv_heads: int, head_dim: int, pages: int, page_size: int, max_pages: int,
                  dtype="float16", cache_dtype=None) -> KernelAdapter:
    """The cache read back: ``k, v = kernel(KCache, VCache[, KScale, VScale], PageTable, Starts)``, each ``[tokens, kv_heads,
    head_dim]`` (one tensor ``[2, ...]``): rows ``Starts[b] .. Starts[b + 1] - 1`` are the first tokens of sequence ``b``, whose
    pages ``PageTable`` int32 ``[sequences, max_pages]`` names in order; ``Starts`` int32 ``[sequences + 1]`` ascending.  Rows of
    no sequence, and tokens whose page is outside of the cache, are zeros.
    """
    fn = "kv_cache_read"
    _positive(fn, sequences=sequences, tokens=tokens, max_pages=max_pages)
    pool = _Pool(fn, kv_heads, head_dim, pages, page_size, dtype, cache_dtype)
    _heads(fn, tokens, kv_heads)
    n = len(pool.params)
    params = [*pool.params, KernelParam("PageTable", torch.int32, (sequences, max_pages)), KernelParam("Starts", torch.int32, (sequences + 1,)),
              KernelParam("kv", pool.dtype, (2, tokens, kv_heads, head_dim))]
    return _kernel(fn, "call_kv_cache_read", params, [n + 2], (*pool.slots(0), n, n + 1, n + 2),
                   (sequences, tokens, kv_heads, head_dim, pages, page_size, max_pages, *pool.ints))


def paged_attention_decode(sequences: int, heads: int, kv_heads: int, head_dim: int, pages: int, page_size: int, max_pages: int,
                           dtype="float16", cache_dtype=None, scale: float | None = None, window: int = 0, sinks: bool = False,
                           with_lse: bool = False) -> KernelAdapter:
    """Attention of one new token a sequence over its cached tokens:
    ``out[, lse] = kernel(q, KCache, VCache[, KScale, VScale], PageTable, Lengths[, Sinks])``, ``q`` and ``out`` ``[sequences, heads,
    head_dim]``, ``Lengths`` int32 ``[sequences]`` counts a sequence's tokens (the new one among them, once it is written).

    Query head ``h`` reads key-value head ``h // (heads // kv_heads)``; ``scale`` is ``head_dim ** -0.5`` by default; ``window`` lets a
    token see the last ``window`` tokens only; ``Sinks`` fp32 ``[heads]`` is one more score a head, whose value is nothing.
    ``with_lse`` also returns fp32 ``[sequences, heads]``, the logarithm of the sum of the scores' exponentials, by which results
    over parts of a context are joined.  A sequence of no tokens gives zeros (and -inf, or the sink).  Softmax and sums are
    fp32; a call gives the same bits every time.
    """
    fn = "paged_attention_decode"
    _positive(fn, sequences=sequences, heads=heads, max_pages=max_pages)
    pool = _Pool(fn, kv_heads, head_dim, pages, page_size, dtype, cache_dtype)
    if heads % kv_heads:
        raise ValueError(f"{fn}: heads={heads} must be a multiple of kv_heads={kv_heads}")
    if head_dim not in ATTENTION_HEAD_DIMS:
        raise ValueError(f"{fn}: head_dim={head_dim} must be one of {ATTENTION_HEAD_DIMS}")
    if heads > 65535 or sequences > attention_sequences(heads, kv_heads, max_pages * page_size):
        raise ValueError(f"{fn}: {sequences} sequences of {heads} heads and up to {max_pages * page_size} tokens: more than a call takes, at most "
                         f"{attention_sequences(heads, kv_heads, max_pages * page_size)} sequences and 65535 heads")
    if window < 0:
        raise ValueError(f"{fn}: window={window} must be 0 (none) or positive")
    window = min(window, max_pages * page_size)  # (32 bits in the library)
    scale = head_dim**-0.5 if scale is None else float(scale)
    if not math.isfinite(scale):
        raise ValueError(f"{fn}: scale must be finite")
    n = 1 + len(pool.params)
    params = [KernelParam("q", pool.dtype, (sequences, heads, head_dim)), *pool.params,
              KernelParam("PageTable", torch.int32, (sequences, max_pages)), KernelParam("Lengths", torch.int32, (sequences,))]
    if sinks:
        params.append(KernelParam("Sinks", torch.float32, (heads,)))
    out = len(params)
    params.append(KernelParam("out", pool.dtype, (sequences, heads, head_dim)))
    if with_lse:
        params.append(KernelParam("lse", torch.float32, (sequences, heads)))
    room = int(_lib.load_library().dq_paged_attention_workspace_bytes(sequences, heads, kv_heads, head_dim, page_size, max_pages, window, pool.ints[1]))
    if room:
        params.append(KernelParam("Workspace", torch.uint8, (room,)))
    slots = (0, *pool.slots(1), n, n + 1, n + 2 if sinks else None, out, out + 1 if with_lse else None, len(params) - 1 if room else None)
    ints = (sequences, heads, kv_heads, head_dim, pages, page_size, max_pages, window, *pool.ints)
    return _kernel(fn, "call_paged_attention_decode", params, [out, out + 1] if with_lse else [out], slots, ints, scale, room,
                   [len(params) - 1] if room else [])
