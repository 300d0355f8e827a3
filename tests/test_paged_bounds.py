"""CPU: the bounds of the paged attention's tests of single weights reject what they are there for."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from tests._paged_ref import f64
from tests._paged_weights import marked, one_above_a_tail, opposite_roundings, weight_bound


def _weights(batch):
    """The last row's weights of sequence 0, first head, in fp64, largest 1; and its values."""

    k, v = batch.rows(f64(batch.k), 0, 0), batch.rows(f64(batch.v), 0, 0)
    row = batch.new[0] - 1
    s = f64(batch.q)[row, 0] @ k.T * batch.scale
    return row, np.exp(s - s.max()), v


def _rejected(batch, out, row):
    want, size = batch.want()
    off = np.abs(out - want[row, 0])
    return bool((off > weight_bound(batch, want, size)[row, 0]).any())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("edges", [False, True])
@pytest.mark.parametrize("new,kv", [([4], [40000]), ([40], [40000]), ([600], [9000])])
def test_one_window_left_out_is_rejected(dtype, dim, edges, new, kv):
    batch = marked(new, kv, edges, heads=1, kv_heads=1, dim=dim, dtype=dtype)
    row, p, v = _weights(batch)
    want, size = batch.want()
    bound = weight_bound(batch, want, size)[row, 0]
    assert (np.abs(p @ v / p.sum() - want[row, 0]) <= bound).all()
    for lost in (slice(0, 64), slice(10048, 10112) if kv[0] > 10112 else slice(4096, 4160), slice(kv[0] - 64, kv[0])):
        q = p.copy()
        q[lost] = 0.0
        assert (np.abs(q @ v / q.sum() - want[row, 0]) > bound).any(), lost
    if edges:
        for lost in (64, 127, kv[0] // 64 * 64 - 1):
            q = p.copy()
            q[lost] = 0.0
            assert (np.abs(q @ v / q.sum() - want[row, 0]) > bound).any(), lost


def test_weights_below_the_smallest_step_are_rejected():
    """The tail in fp16 weights of at most 1, the sum of the same rounded weights."""

    for gap in (24.5, 25.0, 28.25):
        for new in ([1], [40]):
            batch = one_above_a_tail(new, [40000], 5, gap, heads=1, kv_heads=1, dim=64, dtype=torch.float16)
            row, p, v = _weights(batch)
            rounded = f64(torch.from_numpy(p).half())
            assert _rejected(batch, rounded @ v / rounded.sum(), row)
            scaled = f64(torch.from_numpy(p * 2.0**11).half())
            assert new == [1] or not _rejected(batch, scaled @ v / scaled.sum(), row)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_rounded_weights_of_few_rows_are_rejected(dtype):
    for new in ([1], [33]):
        batch = opposite_roundings(new, [500], heads=1, kv_heads=1, dim=64, dtype=dtype)
        row, p, v = _weights(batch)
        rounded = f64(torch.from_numpy(p).to(dtype))
        assert _rejected(batch, rounded @ v / rounded.sum(), row) == (new == [1])
        both = rounded + f64(torch.from_numpy(p - rounded).to(dtype))
        assert not _rejected(batch, both @ v / p.sum(), row)
