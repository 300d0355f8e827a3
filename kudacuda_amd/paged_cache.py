"""A paged KV cache: the pools on the GPU, the bookkeeping of their pages on the host.

One pool tensor ``[2 * layers, num_pages, kv_heads, page_size, head_dim]`` holds
every layer's keys (row 2 l) and values (row 2 l + 1).  A sequence is a list of page
ids and a length; a page may belong to several sequences (``fork``) and is copied
(``kudacuda_copy_pages``) before one of them writes into it.  ``compact`` moves the
pages in use to the lowest ids.  A round of a server is::

    batch = cache.extend([a, b, c], [17, 1, 1])      # slots, tables and lengths of the new tokens
    for layer in range(layers):
        q, k, v = ...                                # projections of the batch's tokens
        q = cache.append(layer, batch, q, k, v, inv_freq)
        out = cache.attend(layer, batch, q)

Calls run on the torch stream that is current when they are made.  The pool is shared
by all of them: a program with several streams orders them itself (events), and a
batch whose calls a graph has captured is kept as long as the graph.
"""

from __future__ import annotations

import math
from dataclasses import dataclass
from typing import Any, Sequence

import numpy as np

from ._native import Native


class OutOfPages(RuntimeError):
    """The pool has too few free pages for the request; nothing was changed."""


@dataclass
class Batch:
    """The new tokens of one round: what append and attend need on the device."""

    sequences: tuple[int, ...]
    tokens: int
    max_query_len: int
    max_kv_len: int
    slots: Any         # int64 [tokens]
    positions: Any     # int32 [tokens]
    query_starts: Any  # int32 [sequences + 1]
    kv_lens: Any       # int32 [sequences]
    page_table: Any    # int32 [sequences, pages of the longest]
    stream: int = 0    # the stream that they were made on


@dataclass
class _Entry:
    pages: list[int]
    length: int


class PagedKvCache:
    """Pages of several sequences in one pool, and the native calls on them."""

    def __init__(self, native: Native, torch: Any, *, layers: int, kv_heads: int, head_dim: int, num_pages: int,
                 page_size: int = 16, dtype: Any = None, device: Any = "cuda:0") -> None:
        dtype = torch.bfloat16 if dtype is None else dtype
        if dtype not in (torch.bfloat16, torch.float16):
            raise ValueError("a cache holds bfloat16 or float16")
        if page_size < 1 or page_size > 4096 or page_size & (page_size - 1) != 0:
            raise ValueError("page_size must be a power of two, 1..4096")
        if min(layers, kv_heads, head_dim, num_pages) < 1 or head_dim % 8 != 0:
            raise ValueError("layers, kv_heads and num_pages must be positive, head_dim a multiple of 8")
        place = torch.device(device)
        if isinstance(native, Native):
            index = torch.cuda.current_device() if place.type == "cuda" and place.index is None else place.index
            if place.type != "cuda" or index != native.device_id:
                raise ValueError(f"a cache on {place} needs a handle of that GPU, not of cuda:{native.device_id}")
        self.native = native
        self.torch = torch
        self.layers = int(layers)
        self.kv_heads = int(kv_heads)
        self.head_dim = int(head_dim)
        self.num_pages = int(num_pages)
        self.page_size = int(page_size)
        self.pool = torch.zeros((2 * layers, num_pages, kv_heads, page_size, head_dim), dtype=dtype, device=device)
        self.device = self.pool.device  # with its number, whichever device is current later
        self._free = list(range(num_pages - 1, -1, -1))  # taken from the end: lowest first
        self._users = [0] * num_pages
        self._entries: dict[int, _Entry] = {}
        self._next = 0
        self._workspaces: dict[Any, Any] = {}

    # ------------------------------------------------------------ bookkeeping
    @property
    def free_pages(self) -> int:
        return len(self._free)

    def length(self, sequence: int) -> int:
        return self._entry(sequence).length

    def pages(self, sequence: int) -> list[int]:
        return list(self._entry(sequence).pages)

    def keys(self, layer: int) -> Any:
        return self.pool[2 * layer]

    def values(self, layer: int) -> Any:
        return self.pool[2 * layer + 1]

    def create(self) -> int:
        """A new, empty sequence."""

        self._entries[self._next] = _Entry([], 0)
        self._next += 1
        return self._next - 1

    def fork(self, sequence: int) -> int:
        """A new sequence with the same tokens; the pages are shared until one of the two writes into them."""

        entry = self._entry(sequence)
        for page in entry.pages:
            self._users[page] += 1
        new = self.create()
        self._entries[new] = _Entry(list(entry.pages), entry.length)
        return new

    def free(self, sequence: int) -> None:
        """Forget a sequence; pages that no other one uses are free again."""

        entry = self._entry(sequence)
        del self._entries[sequence]
        self._drop(entry.pages)

    def truncate(self, sequence: int, length: int) -> None:
        """Forget the tokens from ``length`` on (a rejected draft)."""

        entry = self._entry(sequence)
        if not 0 <= length <= entry.length:
            raise ValueError("a sequence can only become shorter")
        keep = -(-length // self.page_size)
        self._drop(entry.pages[keep:])
        del entry.pages[keep:]
        entry.length = length

    def extend(self, sequences: Sequence[int], counts: Sequence[int]) -> Batch:
        """Room for ``counts[i]`` new tokens behind sequence ``sequences[i]`` each.

        A last page that is shared and has room is copied first.  Raises
        ``OutOfPages`` where the pool is too small.  Where it raises, that or what the
        copy or the batch's upload meets, nothing is changed."""

        sequences = [int(s) for s in sequences]
        counts = [int(c) for c in counts]
        if len(sequences) != len(counts) or not sequences or len(set(sequences)) != len(sequences):
            raise ValueError("one count for each of one or more different sequences")
        if min(counts) < 0 or sum(counts) == 0:
            raise ValueError("counts must not be negative, nor all zero")
        entries = [self._entry(s) for s in sequences]
        size = self.page_size
        # a shared last page is copied by every writer but the last user of it
        users: dict[int, int] = {}
        copied = []
        wanted = 0
        for entry, count in zip(entries, counts):
            page = entry.pages[-1] if count > 0 and entry.length % size != 0 else None
            copy = page is not None and users.setdefault(page, self._users[page]) > 1
            if copy:
                users[page] -= 1
            copied.append(copy)
            wanted += -(-(entry.length + count) // size) - len(entry.pages) + copy
        if wanted > len(self._free):
            raise OutOfPages(f"{wanted} pages wanted, {len(self._free)} free")
        before = [(entry.length, len(entry.pages), entry.pages[-1:]) for entry in entries]
        shared = {page: self._users[page] for page in users}
        left = len(self._free) - wanted
        fresh = self._free[left:]
        pairs = []
        try:
            for entry, count, copy in zip(entries, counts, copied):
                if copy:
                    page = self._take()
                    pairs.append((entry.pages[-1], page))
                    self._users[entry.pages[-1]] -= 1
                    entry.pages[-1] = page
                entry.length += count
                while len(entry.pages) * size < entry.length:
                    entry.pages.append(self._take())
            batch = self._batch(sequences, entries, counts)
            self._copy(pairs)
            return batch
        except BaseException:
            for entry, (length, n, last) in zip(entries, before):
                entry.length = length
                entry.pages[max(0, n - 1):] = last
            for page, n in [*shared.items(), *((page, 0) for page in fresh)]:
                self._users[page] = n
            self._free[left:] = fresh
            raise

    def compact(self) -> int:
        """Move the pages in use to the lowest ids (the pool could then be cut); returns how many moved.

        Batches made before name the old pages and must not be used any more."""

        used = [p for p in range(self.num_pages) if self._users[p] > 0]
        low = [p for p in range(len(used)) if self._users[p] == 0]
        moves = dict(zip([p for p in used if p >= len(used)], low))
        self._copy(list(moves.items()))
        for entry in self._entries.values():
            entry.pages = [moves.get(p, p) for p in entry.pages]
        for old, new in moves.items():
            self._users[new], self._users[old] = self._users[old], 0
        self._free = list(range(self.num_pages - 1, len(used) - 1, -1))
        return len(moves)

    def _entry(self, sequence: int) -> _Entry:
        if sequence not in self._entries:
            raise KeyError(f"no sequence {sequence}")
        return self._entries[sequence]

    def _take(self) -> int:
        page = self._free.pop()
        self._users[page] = 1
        return page

    def _drop(self, pages: Sequence[int]) -> None:
        for page in pages:
            self._users[page] -= 1
            if self._users[page] == 0:
                self._free.append(page)
        self._free.sort(reverse=True)

    def _batch(self, sequences, entries, counts) -> Batch:
        t, size = self.torch, self.page_size
        table = np.zeros((len(entries), max(1, max(len(e.pages) for e in entries))), dtype=np.int32)
        positions = []
        slots = []
        for row, entry, count in zip(table, entries, counts):
            row[:len(entry.pages)] = entry.pages
            at = np.arange(entry.length - count, entry.length)
            positions.append(at)
            slots.append(row[at // size].astype(np.int64) * size + at % size)
        lengths = np.array([e.length for e in entries], dtype=np.int32)
        starts = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)

        def up(a: np.ndarray) -> Any:
            return t.from_numpy(np.ascontiguousarray(a)).to(self.device)

        return Batch(tuple(sequences), int(starts[-1]), max(counts), int(lengths.max()), up(np.concatenate(slots)),
                     up(np.concatenate(positions).astype(np.int32)), up(starts), up(lengths), up(table), self._stream())

    # ------------------------------------------------------------ native calls
    def _stream(self) -> int:
        return self.torch.cuda.current_stream(self.device).cuda_stream

    def _dtype(self) -> int:
        return 1 if self.pool.dtype == self.torch.bfloat16 else 2

    def _capturing(self) -> bool:
        """Whether a graph captures the current stream of the cache's device."""

        cuda = self.torch.cuda
        if cuda.current_device() == self.device.index:
            return cuda.is_current_stream_capturing()
        with cuda.device(self.device):
            return cuda.is_current_stream_capturing()

    def _use(self, batch: Batch) -> tuple[int, bool]:
        """The current stream, and whether it is captured; where the batch was made on another one, its memory waits
        for this one too."""

        stream, capturing = self.torch.cuda.current_stream(self.device), self._capturing()
        if stream.cuda_stream != batch.stream and not capturing:
            for x in (batch.slots, batch.positions, batch.query_starts, batch.kv_lens, batch.page_table):
                x.record_stream(stream)
        return stream.cuda_stream, capturing

    def _copy(self, pairs: Sequence[tuple[int, int]]) -> None:
        if not pairs:
            return
        pool = self.pool
        table = np.ascontiguousarray(pairs, dtype=np.int32)
        size = pool.element_size()
        self.native.call("kudacuda_copy_pages", pool.data_ptr(), table.ctypes.data, len(table), pool.shape[0],
                         self.num_pages, pool.stride(1) * size, pool.stride(1) * size, pool.stride(0) * size,
                         self._stream())

    def _rows(self, name: str, x: Any, tokens: int, heads: int | None) -> int:
        """Check [tokens, heads, head_dim] rows with packed heads; returns the stride between tokens."""

        if (x.dim() != 3 or x.shape[0] != tokens or (heads is not None and x.shape[1] != heads)
                or x.shape[2] != self.head_dim or x.dtype != self.pool.dtype or x.device != self.pool.device):
            raise ValueError(f"{name} must be [{tokens}, {heads or 'heads'}, {self.head_dim}] {self.pool.dtype} "
                             f"on {self.pool.device}")
        if x.stride(2) != 1 or (x.shape[1] > 1 and x.stride(1) != self.head_dim):
            raise ValueError(f"the heads of a token of {name} must be contiguous")
        return x.stride(0) if tokens > 1 else x.shape[1] * self.head_dim

    def append(self, layer: int, batch: Batch, query: Any, key: Any, value: Any, inv_freq: Any, *,
               amplitude: float = 1.0, interleaved: bool = False, out: Any = None) -> Any:
        """Turn ``query`` and ``key`` at the batch's positions, write keys and values into the pages; returns the
        turned queries (``out``, which may be ``query``).  ``inv_freq``: float64 on the device, half of the
        rotated dims."""

        q_stride = self._rows("query", query, batch.tokens, None)
        k_stride = self._rows("key", key, batch.tokens, self.kv_heads)
        v_stride = self._rows("value", value, batch.tokens, self.kv_heads)
        if inv_freq.dtype != self.torch.float64 or inv_freq.device != self.pool.device or not inv_freq.is_contiguous():
            raise ValueError("inv_freq must be contiguous float64 on the cache's device")
        out = self.torch.empty_like(query, memory_format=self.torch.contiguous_format) if out is None else out
        o_stride = self._rows("out", out, batch.tokens, query.shape[1])
        keys, values = self.keys(layer), self.values(layer)
        stream, _ = self._use(batch)
        self.native.call("kudacuda_rope_paged_append", query.data_ptr(), key.data_ptr(), value.data_ptr(),
                         inv_freq.data_ptr(), batch.positions.data_ptr(), batch.slots.data_ptr(), out.data_ptr(),
                         keys.data_ptr(), values.data_ptr(), self._dtype(), batch.tokens, query.shape[1],
                         self.kv_heads, self.head_dim, 2 * inv_freq.numel(), int(interleaved), q_stride, k_stride,
                         v_stride, o_stride, self.num_pages, self.page_size, keys.stride(0), keys.stride(1),
                         keys.stride(2), float(amplitude), stream)
        return out

    def attend(self, layer: int, batch: Batch, query: Any, *, scale: float | None = None, out: Any = None) -> Any:
        """Causal attention of the batch's new tokens over their sequences; returns [tokens, heads, head_dim]."""

        q_stride = self._rows("query", query, batch.tokens, None)
        heads = query.shape[1]
        out = self.torch.empty_like(query, memory_format=self.torch.contiguous_format) if out is None else out
        o_stride = self._rows("out", out, batch.tokens, heads)
        keys, values = self.keys(layer), self.values(layer)
        n = len(batch.sequences)
        nbytes = self.native.lib.kudacuda_paged_attention_workspace_bytes(
            batch.tokens, n, batch.max_query_len, batch.max_kv_len, heads, self.kv_heads, self.head_dim)
        stream, capturing = self._use(batch)
        # a workspace a stream: calls on one stream follow one another; a captured call
        # gets its own, from its graph's memory
        workspace = None if capturing else self._workspaces.get(stream)
        if nbytes > 0 and (workspace is None or workspace.numel() < nbytes):
            workspace = self.torch.empty(nbytes, dtype=self.torch.uint8, device=self.device)
            if not capturing:
                self._workspaces[stream] = workspace
        self.native.call("kudacuda_paged_attention", query.data_ptr(), keys.data_ptr(), values.data_ptr(),
                         batch.page_table.data_ptr(), batch.query_starts.data_ptr(), batch.kv_lens.data_ptr(),
                         out.data_ptr(), workspace.data_ptr() if nbytes > 0 else 0, nbytes, self._dtype(),
                         batch.tokens, n, batch.max_query_len, batch.max_kv_len, heads, self.kv_heads, self.head_dim,
                         q_stride, o_stride, self.num_pages, self.page_size, batch.page_table.shape[1],
                         keys.stride(0), keys.stride(1), keys.stride(2),
                         1.0 / math.sqrt(self.head_dim) if scale is None else float(scale), stream)
        return out
