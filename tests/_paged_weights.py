"""Batches over a paged cache that show what attention does with single weights (test infrastructure): inputs whose
rounding or loss of a weight adds up instead of averaging out."""

from __future__ import annotations

import numpy as np
import torch

from tests._paged_ref import HALF, Paged

LN2 = float(np.float32(np.log(2.0)))
# Weights of sequences of which a KV head has at most so many rows keep two 16-bit parts.
FINE_ROWS = 32


def fine_rows(batch: Paged) -> np.ndarray:
    """Which of the batch's rows belong to sequences of few rows."""

    group = batch.heads // batch.kv_heads
    return np.concatenate([np.full(n, n * group <= FINE_ROWS) for n in batch.new])


def told(batch: Paged, hint: int | None) -> Paged:
    """The longest length that the batch's calls are told, and a table as wide: what is told counts up to a row of it."""

    batch.hint = hint
    if hint is not None:
        table = np.full((len(batch.kv), -(-hint // batch.page)), -7, dtype=np.int32)
        table[:, :batch.table.shape[1]] = batch.table
        batch.table = table
    return batch


def weight_bound(batch: Paged, want: np.ndarray, size: np.ndarray) -> np.ndarray:
    """How far an output may be off where scores are small (below 2^5 after the scale): half a step of its type (and
    of the type's smallest step), and of size = sum |weight * value|
      * fp32: a score is off by 2 roundings of 2^5 at most, 2^-18, and with exp2 and the sums of up to 2^10 products
        of the matrix instructions, 2^-24 each at worst, below 2^-13;
      * the weights' own rounding: half a step of the type, or, in two parts, the second part's half step of a half
        step, 2^-16 (bf16) or less;
    and in fp16, whose weights are scaled into the type's upper range, half of its smallest step, 2^-25, of 2^11 at
    least: 2^-36 a key of the largest weight, which is 1, times the largest value."""

    half = HALF[batch.dtype]
    coarse = np.where(fine_rows(batch), 2.0**-16, half)[:, None, None]
    bound = half * np.abs(want) + (2.0**-13 + coarse) * size
    if batch.dtype == torch.float16:
        top = float(batch.v[~torch.isnan(batch.v)].abs().max())
        bound += 2.0**-25 + max(batch.kv) * 2.0**-36 * top
    return bound


def _place(batch: Paged, i: int, key: int) -> tuple[int, int]:
    return int(batch.table[i, key // batch.page]), key % batch.page


def _clear(batch: Paged, value: float) -> None:
    """Queries of one in the first dim, keys of zero, values of `value`; what no sequence has stays NaN."""

    batch.q.zero_()
    batch.q[..., 0] = 1.0
    nan = torch.isnan(batch.k)
    batch.k = torch.where(nan, batch.k, torch.zeros_like(batch.k))
    batch.v = torch.where(nan, batch.v, torch.full_like(batch.v, value))


def one_above_a_tail(new, kv, key: int, gap: float, **kwargs) -> Paged:
    """Key `key` of every sequence has 2^gap times the weight of each other one and no value, the others have 1: the
    result is the tail's share."""

    batch = Paged(31, new, kv, scale=LN2, **kwargs)
    _clear(batch, 1.0)
    for i, n in enumerate(kv):
        page, at = _place(batch, i, min(key, n - 1))
        batch.k[page, :, at, 0] = gap
        batch.v[page, :, at] = 0.0
    return batch


def opposite_roundings(new, kv, **kwargs) -> Paged:
    """Two weights that the type rounds in opposite directions, with values that cancel, and every 16th key of the
    largest weight and no value: a rounded weight shows in full."""

    batch = Paged(32, new, kv, scale=LN2, **kwargs)
    _clear(batch, 0.0)
    steps = torch.arange(-384, -2, dtype=torch.float32) / 128  # exact in both types
    weights = torch.exp2(steps.double())
    off = (weights.to(batch.dtype).double() - weights) / weights
    down, up = int(off.argmin()), int(off.argmax())
    value = float((weights[down] / weights[up]).to(batch.dtype))
    for i, n in enumerate(kv):
        j = np.arange(n)
        pages, at = batch.table[i, j // batch.page], j % batch.page
        for which, step, v in ((j % 16 != 0) & (j % 2 == 0), steps[down], 1.0), ((j % 2 == 1), steps[up], -value):
            rows = torch.from_numpy(pages[which].astype(np.int64)), slice(None), torch.from_numpy(at[which])
            batch.k[rows[0], :, rows[2], 0] = float(step)
            batch.v[rows[0], :, rows[2]] = v
    return batch


def marked(new, kv, edges: bool, **kwargs) -> Paged:
    """Scores that are nearly equal; a value of 1 in dim (window of 64 keys) modulo dim, at every key of the window or
    (edges) at its first and last alone: each window, or each of these keys, is a visible share of its dim."""

    batch = Paged(33, new, kv, scale=0.02, **kwargs)
    batch.v = torch.where(torch.isnan(batch.v), batch.v, torch.zeros_like(batch.v))
    for i, n in enumerate(kv):
        j = np.arange(n)
        j = j[(j % 64 == 0) | (j % 64 == 63)] if edges else j
        pages = torch.from_numpy(batch.table[i, j // batch.page].astype(np.int64))
        batch.v[pages, :, torch.from_numpy(j % batch.page), torch.from_numpy(j // 64 % batch.dim)] = 1.0
    return batch
