"""Low-rank adapters of many requests beside a shared projection.

A server that shares one NF4 model between requests keeps, for every projection that its
adapters change, their factors on the GPU (``LoraAdapters``), and says once a round which
rows belong to which adapter (``lora_batch``)::

    adapters = LoraAdapters(native, torch, in_features=2048, out_features=11008, adapters=64, max_rank=64)
    adapters.load(3, a, b, scale=alpha / rank)       # a [rank, in], b [out, rank]
    batch = lora_batch(torch, [3, None, 7], [1, 1, 300])  # adapters of three requests, and their rows
    y = ...                                          # the shared projection of x
    adapters.add(batch, x, y)                        # y += scale * (x a^T) b^T, request by request

Calls run on the torch stream that is current when they are made.
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import Any, Sequence

import numpy as np

from ._native import Native

TILE = 64  # rows of a tile at most
MAX_RANK = 128


@dataclass
class LoraBatch:
    """Which rows of a round belong to which adapter: rows in the adapters' order, and tiles of one adapter's rows."""

    tokens: int
    tile_count: int
    order: Any       # int32 [tokens]
    tiles: Any       # int32 [tiles, 3]: adapter (-1: none), first of order, how many
    stream: int = 0  # the stream that they were made on
    most: int = -1   # the largest adapter


def lora_batch(torch: Any, adapters: Sequence[int | None], counts: Sequence[int], device: Any = "cuda:0") -> LoraBatch:
    """The plan of a round: request i has ``counts[i]`` rows, one after the other, and adapter ``adapters[i]``."""

    counts = [int(c) for c in counts]
    of = [-1 if a is None else int(a) for a in adapters]
    if len(of) != len(counts) or not of or min(counts) < 0 or sum(counts) == 0 or min(of) < -1:
        raise ValueError("one adapter (or None) and one count for each of one or more requests, not all counts zero")
    rows = np.repeat(np.asarray(of, dtype=np.int64), counts)
    order = np.argsort(rows, kind="stable").astype(np.int32)
    names, first, many = np.unique(rows[order], return_index=True, return_counts=True)
    tiles = [(a, f + i, min(TILE, n - i)) for a, f, n in zip(names, first, many) for i in range(0, n, TILE)]
    table = np.asarray(tiles, dtype=np.int32)
    device = torch.device(device)
    stream = torch.cuda.current_stream(device).cuda_stream if device.type == "cuda" else 0
    return LoraBatch(len(rows), len(table), torch.from_numpy(order).to(device), torch.from_numpy(table).to(device), stream,
                     max(of))


class LoraAdapters:
    """The factors of one projection's adapters, and the native call on them."""

    def __init__(self, native: Native, torch: Any, *, in_features: int, out_features: int, adapters: int, max_rank: int,
                 dtype: Any = None, device: Any = "cuda:0") -> None:
        dtype = torch.bfloat16 if dtype is None else dtype
        if dtype not in (torch.bfloat16, torch.float16):
            raise ValueError("adapters hold bfloat16 or float16")
        if not 1 <= max_rank <= MAX_RANK or not 1 <= adapters <= 65536:
            raise ValueError(f"ranks up to {MAX_RANK} and 1..65536 adapters")
        if min(in_features, out_features) < 8 or in_features % 8 != 0 or out_features % 8 != 0:
            raise ValueError("in_features and out_features must be multiples of 8")
        place = torch.device(device)
        if isinstance(native, Native):
            index = torch.cuda.current_device() if place.type == "cuda" and place.index is None else place.index
            if place.type != "cuda" or index != native.device_id:
                raise ValueError(f"adapters on {place} need a handle of that GPU, not of cuda:{native.device_id}")
        self.native = native
        self.torch = torch
        self.in_features = int(in_features)
        self.out_features = int(out_features)
        self.count = int(adapters)
        self.max_rank = -(-int(max_rank) // 8) * 8
        self.dtype = dtype
        self.a = torch.zeros((adapters, self.max_rank, in_features), dtype=dtype, device=device)
        self.b = torch.zeros((adapters, out_features * self.max_rank), dtype=dtype, device=device)
        self.ranks = torch.zeros(adapters, dtype=torch.int32, device=device)
        self.scales = torch.zeros(adapters, dtype=torch.float32, device=device)
        self.device = self.a.device  # with its number, whichever device is current later

    def _index(self, index: int) -> int:
        if not 0 <= index < self.count:
            raise IndexError(f"adapter {index} of {self.count}")
        return index

    def load(self, index: int, a: Any, b: Any, scale: float = 1.0) -> None:
        """Adapter ``index`` becomes ``a`` [rank, in_features], ``b`` [out_features, rank] and ``scale``."""

        index, rank = self._index(index), a.shape[0]
        if (a.dim() != 2 or b.dim() != 2 or not 1 <= rank <= self.max_rank or a.shape[1] != self.in_features
                or tuple(b.shape) != (self.out_features, rank)):
            raise ValueError(f"factors must be [rank, {self.in_features}] and [{self.out_features}, rank], rank 1.."
                             f"{self.max_rank}")
        a, b = a.detach(), b.detach()
        pitch = -(-rank // 8) * 8
        rows = self.torch.zeros((self.out_features, pitch), dtype=self.dtype, device=self.device)
        rows[:, :rank] = b
        self.a[index, :rank] = a
        self.b[index, :rows.numel()] = rows.view(-1)
        self.ranks[index] = rank
        self.scales[index] = float(scale)

    def clear(self, index: int) -> None:
        """Adapter ``index`` adds nothing any more."""

        self.ranks[self._index(index)] = 0

    def _rows(self, name: str, x: Any, tokens: int, features: int) -> int:
        """Check [tokens, features] rows; returns the stride between them."""

        if (x.dim() != 2 or x.shape[0] != tokens or x.shape[1] != features or x.dtype != self.dtype
                or x.device != self.device):
            raise ValueError(f"{name} must be [{tokens}, {features}] {self.dtype} on {self.device}")
        if x.stride(1) != 1:
            raise ValueError(f"the rows of {name} must be contiguous")
        return x.stride(0) if tokens > 1 else features

    def _capturing(self) -> bool:
        cuda = self.torch.cuda
        if cuda.current_device() == self.device.index:
            return cuda.is_current_stream_capturing()
        with cuda.device(self.device):
            return cuda.is_current_stream_capturing()

    def add(self, batch: LoraBatch, x: Any, base: Any, out: Any = None) -> Any:
        """``out`` = ``base`` + what every row's adapter makes of ``x``; ``out`` is ``base`` unless given."""

        out = base if out is None else out
        if batch.most >= self.count:
            raise IndexError(f"adapter {batch.most} of {self.count}")
        if batch.order.device != self.device:
            raise ValueError(f"a plan on {batch.order.device} for adapters on {self.device}")
        x_stride = self._rows("x", x, batch.tokens, self.in_features)
        base_stride = self._rows("base", base, batch.tokens, self.out_features)
        out_stride = self._rows("out", out, batch.tokens, self.out_features)
        stream, capturing = self.torch.cuda.current_stream(self.device), self._capturing()
        if stream.cuda_stream != batch.stream and not capturing:
            for rows in (batch.order, batch.tiles):
                rows.record_stream(stream)
        nbytes = self.native.lib.kudacuda_lora_workspace_bytes(batch.tokens, batch.tile_count, self.max_rank,
                                                               self.in_features)
        # a workspace a stream for all adapters of the handle: calls on one stream follow one
        # another; a captured call gets its own, from its graph's memory
        shared, use = self.native.workspaces, ("adapters", stream.cuda_stream)
        workspace = None if capturing else shared.get(use)
        if workspace is None or workspace.numel() < nbytes:
            workspace = self.torch.empty(nbytes, dtype=self.torch.uint8, device=self.device)
            if not capturing:
                shared[use] = workspace
        self.native.call("kudacuda_lora_add", x.data_ptr(), self.a.data_ptr(), self.b.data_ptr(), self.ranks.data_ptr(),
                         self.scales.data_ptr(), batch.order.data_ptr(), batch.tiles.data_ptr(), base.data_ptr(),
                         out.data_ptr(), workspace.data_ptr(), nbytes, 1 if self.dtype == self.torch.bfloat16 else 2,
                         batch.tokens, batch.tile_count, self.count, self.max_rank, self.in_features, self.out_features,
                         x_stride, base_stride, out_stride, stream.cuda_stream)
        return out
