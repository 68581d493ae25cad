"""The attention of a decoder block on the kernels: :class:`PagedKVCache`, and :class:`W4Attention` between two
:class:`~tilelang_amd.w4linear.W4A16Linear` projections.

A step has rows: the new tokens of every sequence, one sequence behind the other.  One token a sequence is a decode step; several
are a prompt or a part of one, and each of them sees the tokens before it and itself.  ``rows = cache.extend(counts)`` finds their
places once for all layers, ``layer(x, cache, rows)`` projects, rotates and writes, attends and projects back.

The attention is that of one new token: every row reads its whole context, so a prompt of n tokens reads n / 2 of them n times.
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import Sequence

import torch
from torch import nn

from . import kv_kernels
from .w4linear import W4A16Linear


@dataclass(frozen=True)
class Rows:
    """The new tokens of a step, on the device, a sequence's one behind the other in their order: of each its position, its slot in the
    cache, its sequence's row of the page table and how many tokens it sees.  ``owners``: where a row of ``pages`` for every token would
    take too much memory, ``pages`` has one for every sequence, and this is the one of each token."""

    positions: torch.Tensor
    slots: torch.Tensor
    pages: torch.Tensor
    lengths: torch.Tensor
    owners: torch.Tensor | None = None

    def pages_of(self, part: slice) -> torch.Tensor:
        """The rows of the page table of some of the tokens."""
        return self.pages[part] if self.owners is None else self.pages[self.owners[part]]


#: kernel objects that a cache keeps: prompts come in any number of rows
MAX_KERNELS = 64
#: page ids (256 MiB) of a step's tokens that are held at once
MAX_PAGE_IDS = 2**26


class PagedKVCache:
    """Keys and values of some sequences in ``layers`` layers, in pages that the layers' caches are cut into alike.

    ``cache_dtype``: ``dtype`` itself, ``"float8_e4m3fn"`` or ``"int8"`` (one fp32 scale a token and head).  ``pages`` are shared by
    the sequences as they grow; ``extend`` takes what it needs, or raises and takes nothing, and ``release`` gives a sequence's back.
    ``page_table`` is another tensor after each change, so the :class:`Rows` of a step keep the pages that they were made with.
    """

    def __init__(self, sequences: int, pages: int, kv_heads: int, head_dim: int, page_size: int = 64, max_tokens: int | None = None,
                 layers: int = 1, dtype="float16", cache_dtype=None, device="cuda"):
        pool = kv_kernels._Pool("PagedKVCache", kv_heads, head_dim, pages, page_size, dtype, cache_dtype)
        kv_kernels._positive("PagedKVCache", sequences=sequences, layers=layers)
        max_tokens = pages * page_size if max_tokens is None else max_tokens
        kv_kernels._positive("PagedKVCache", max_tokens=max_tokens)
        self.sequences, self.pages, self.kv_heads, self.head_dim, self.page_size, self.layers = sequences, pages, kv_heads, head_dim, page_size, layers
        self.max_tokens, self.max_pages = max_tokens, -(-max_tokens // page_size)
        self.dtype, self.cache_dtype, self.device = pool.dtype, pool.held, torch.device(device)
        shape = (layers, pages, kv_heads, page_size, head_dim)
        self.keys, self.values = (torch.zeros(shape, dtype=pool.held, device=device) for _ in range(2))
        self.key_scale = self.value_scale = None
        if pool.scaled:
            self.key_scale, self.value_scale = (torch.zeros(shape[:4], dtype=torch.float32, device=device) for _ in range(2))
        self.lengths = [0] * sequences
        self._free = list(range(pages - 1, -1, -1))
        self._pages: list[list[int]] = [[] for _ in range(sequences)]
        self.page_table = torch.full((sequences, self.max_pages), -1, dtype=torch.int32, device=device)
        self._kernels: dict = {}

    def sizes(self) -> dict:
        """What the kernel factories are told about the cache."""
        return dict(kv_heads=self.kv_heads, head_dim=self.head_dim, pages=self.pages, page_size=self.page_size, dtype=self.dtype,
                    cache_dtype=None if self.cache_dtype == self.dtype else str(self.cache_dtype).removeprefix("torch."))

    def pool(self, layer: int = 0) -> tuple:
        """A layer's ``KCache, VCache[, KScale, VScale]``, as the kernel objects take them."""
        pool = (self.keys[layer], self.values[layer])
        return pool if self.key_scale is None else (*pool, self.key_scale[layer], self.value_scale[layer])

    def extend(self, counts: Sequence[int]) -> Rows:
        """Room for ``counts[b]`` new tokens of every sequence ``b``."""
        if len(counts) != self.sequences or any(c < 0 for c in counts) or not any(counts):
            raise ValueError(f"extend: expected {self.sequences} counts that are not negative, some positive (got {list(counts)})")
        wanted = [-(-(n + c) // self.page_size) - len(p) for n, c, p in zip(self.lengths, counts, self._pages)]
        for b, (n, c) in enumerate(zip(self.lengths, counts)):
            if n + c > self.max_tokens:
                raise RuntimeError(f"extend: sequence {b} would have {n + c} tokens, more than max_tokens={self.max_tokens}")
        if sum(wanted) > len(self._free):
            raise RuntimeError(f"extend: {sum(wanted)} pages wanted, {len(self._free)} free")
        changed = [b for b, w in enumerate(wanted) if w]
        for b in changed:
            self._pages[b] += [self._free.pop() for _ in range(wanted[b])]
        if changed:
            rows = torch.tensor([self._pages[b] + [-1] * (self.max_pages - len(self._pages[b])) for b in changed], dtype=torch.int32)
            self.page_table = self.page_table.index_copy(0, torch.tensor(changed, device=self.device), rows.to(self.device))
        positions, slots, owners = [], [], []
        for b, c in enumerate(counts):
            for t in range(self.lengths[b], self.lengths[b] + c):
                positions.append(t)
                slots.append(self._pages[b][t // self.page_size] * self.page_size + t % self.page_size)
                owners.append(b)
            self.lengths[b] += c
        both = torch.tensor([positions, slots], dtype=torch.int32).to(self.device)
        # (one token of every sequence: the table as it stands)
        if owners == list(range(self.sequences)):
            return Rows(both[0], both[1], self.page_table, both[0] + 1)
        owner = torch.tensor(owners, device=self.device)
        if len(owners) * self.max_pages > MAX_PAGE_IDS:
            return Rows(both[0], both[1], self.page_table, both[0] + 1, owner)
        return Rows(both[0], both[1], self.page_table[owner], both[0] + 1)

    def release(self, sequence: int) -> None:
        """The sequence has no tokens any more; its pages are free."""
        self._free += reversed(self._pages[sequence])
        self._pages[sequence], self.lengths[sequence] = [], 0
        self.page_table = self.page_table.clone()
        self.page_table[sequence] = -1

    def read(self, layer: int = 0) -> tuple:
        """Keys and values of all sequences, one behind the other, each ``[tokens, kv_heads, head_dim]`` in ``dtype``."""
        tokens = sum(self.lengths)
        if not tokens:
            empty = torch.empty((0, self.kv_heads, self.head_dim), dtype=self.dtype, device=self.device)
            return empty, empty.clone()
        starts = torch.tensor([0, *self.lengths]).cumsum(0).int().to(self.device)
        kernel = kv_kernels.kv_cache_read(self.sequences, tokens, max_pages=self.max_pages, **self.sizes())
        k, v = kernel(*self.pool(layer), self.page_table, starts)
        return k, v

    def kernel(self, make, *args, **kwargs):
        """The kernel object ``make(*args, **kwargs, **sizes())``, made once for all layers; the last :data:`MAX_KERNELS` used are kept."""
        key = (make, args, tuple(sorted(kwargs.items())))
        found = self._kernels.pop(key, None)
        if found is None:
            found = make(*args, **kwargs, **self.sizes())
            while len(self._kernels) >= MAX_KERNELS:
                del self._kernels[next(iter(self._kernels))]
        self._kernels[key] = found  # (the last in the order)
        return found


class W4Attention(nn.Module):
    """A decoder block's attention in fp16 on 4-bit weights: ``o(attend(rotate(q), cache(rotate(k), v)))`` with one fused projection
    of queries, keys and values.  ``rotary``: the table of :func:`rotary_table` for the positions that the model is run at;
    ``rotary_dim`` and ``interleaved`` as for :func:`rotary`; ``window`` and ``sinks`` as for :func:`paged_attention_decode`."""

    def __init__(self, hidden: int, heads: int, kv_heads: int, head_dim: int, rotary: torch.Tensor, interleaved: bool = False, window: int = 0,
                 sinks: bool = False, scale: float | None = None, group_size: int = 128, with_zeros: bool = False, bias: bool = False):
        super().__init__()
        self.heads, self.kv_heads, self.head_dim = heads, kv_heads, head_dim
        self.interleaved, self.window, self.scale = interleaved, window, scale
        self.qkv = W4A16Linear(hidden, (heads + 2 * kv_heads) * head_dim, group_size=group_size, with_zeros=with_zeros, bias=bias)
        self.o = W4A16Linear(heads * head_dim, hidden, group_size=group_size, with_zeros=with_zeros, bias=bias)
        self.register_buffer("rotary", rotary, persistent=False)
        self.register_buffer("sinks", torch.zeros((heads,), dtype=torch.float32) if sinks else None)

    def _apply(self, fn, *args, **kwargs):
        # The kernels read both in fp32 whatever type a model is turned into, and a table rounded in between has lost its angles: they
        # are moved, not converted.
        kept = {name: b for name in ("rotary", "sinks") if (b := self._buffers[name]) is not None and b.dtype == torch.float32}
        super()._apply(fn, *args, **kwargs)
        for name, b in kept.items():
            if self._buffers[name].dtype != torch.float32:
                self._buffers[name] = b.to(self._buffers[name].device)
        return self

    def attend(self, qkv: torch.Tensor, cache: PagedKVCache, rows: Rows, layer: int = 0) -> torch.Tensor:
        """``qkv`` ``[rows, heads + 2 kv_heads, head_dim]`` -> ``[rows, heads, head_dim]``; its keys and values go into the cache."""
        n, at_once = qkv.shape[0], self._rows_at_once(cache)
        if n <= at_once and rows.owners is None:
            return self._attend(qkv, cache, rows, layer)
        # (a row sees tokens of its own part and of those before it only, as a sequence's rows come in their order)
        parts = [slice(at, min(at + at_once, n)) for at in range(0, n, at_once)]
        return torch.cat([self._attend(qkv[p], cache, Rows(rows.positions[p], rows.slots[p], rows.pages_of(p), rows.lengths[p]), layer) for p in parts])

    def _rows_at_once(self, cache: PagedKVCache) -> int:
        """What one call of the write and of the attention takes."""
        return max(1, min(kv_kernels.attention_sequences(self.heads, self.kv_heads, cache.max_pages * cache.page_size),
                          kv_kernels.MAX_HEADS // (self.heads + 2 * self.kv_heads), MAX_PAGE_IDS // cache.max_pages))

    def _attend(self, qkv: torch.Tensor, cache: PagedKVCache, rows: Rows, layer: int) -> torch.Tensor:
        n, (positions, rotary_dim) = qkv.shape[0], self.rotary.shape
        write = cache.kernel(kv_kernels.rotary_kv_cache_write, n, self.heads, positions=positions, rotary_dim=rotary_dim, interleaved=self.interleaved)
        attend = cache.kernel(kv_kernels.paged_attention_decode, n, self.heads, max_pages=cache.max_pages, window=self.window,
                              sinks=self.sinks is not None, scale=self.scale)
        pool = cache.pool(layer)
        q = write(qkv, self.rotary, rows.positions, rows.slots, *pool)
        return attend(q, *pool, rows.pages, rows.lengths, *(() if self.sinks is None else (self.sinks,)))

    def forward(self, x: torch.Tensor, cache: PagedKVCache, rows: Rows, layer: int = 0) -> torch.Tensor:
        """``x`` ``[rows, hidden]`` -> ``[rows, hidden]``, ``rows`` of ``cache.extend``, the same for every layer of a step."""
        qkv = self.qkv(x).view(x.shape[0], self.heads + 2 * self.kv_heads, self.head_dim)
        return self.o(self.attend(qkv, cache, rows, layer).view(x.shape[0], self.heads * self.head_dim))
