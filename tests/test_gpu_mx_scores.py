"""GPU: scores of attention over a cache of 8 or 4 bits whose queries and keys have dims of very unlike size."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from tests._mx_ref import MxPaged
from tests._paged_ref import f64

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16
every = [pytest.mark.parametrize("hint", [None, 1 << 20]), pytest.mark.parametrize("bits", [4, 8]),
         pytest.mark.parametrize("dtype", [BF16, FP16]),
         pytest.mark.parametrize("new,kv", [([1], [40]), ([1, 2, 1], [300, 7, 1]), ([12, 40], [60, 90])])]


def each_form(test):
    for mark in every:
        test = mark(test)
    return test


def _check(batch, native, off=2.0**-11):
    """Within the batches' bound, whose share for the scores' sums (2^-11 of sum |weight * value|) may be another."""

    want, size = batch.want()
    got = f64(batch.call(native, batch.device()))
    bound = batch.bound(want, size) + (off - 2.0**-11) * size
    assert np.isfinite(got).all()
    assert (np.abs(got - want) <= bound).all(), float((np.abs(got - want) / bound).max())


@each_form
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("apart", [2, 8])
def test_small_dims_beside_large_ones_that_cancel(torch_gpu, native, dtype, bits, dim, new, kv, hint, apart):
    """Pairs of dims of 2^14 cancel, whole numbers of at most 3 beside them decide.  All are numbers of the cache and of
    the type; products are whole and all partial sums below 2 * 32 * 2^16, so sums in fp32 are exact in any order."""

    batch = MxPaged(21, new, kv, bits=bits, dtype=dtype, dim=dim, heads=4, kv_heads=2)
    batch.hint = hint
    rng = np.random.default_rng([5, dim, apart])
    q = rng.integers(-3, 4, batch.q.shape).astype(np.float64)
    k = rng.integers(-3, 4, batch.k.shape).astype(np.float64)
    large = np.arange(0, dim, 2 * apart)
    q[..., large] = q[..., large + apart] = 2.0**14 * rng.choice([-1, 1], (*q.shape[:-1], len(large)))
    k[..., large] = 4 * rng.choice([-1, 1], (*k.shape[:-1], len(large)))
    k[..., large + apart] = -k[..., large]
    batch.q, batch.k = (torch.from_numpy(x).to(dtype) for x in (q, k))
    batch.v = batch.v.nan_to_num(0.0)
    batch.repack()
    assert np.array_equal(f64(batch.k), k)
    _check(batch, native)


@each_form
@pytest.mark.parametrize("dim", [64, 128])
def test_blocks_and_dims_of_unlike_size(torch_gpu, native, dtype, bits, dim, new, kv, hint):
    """Every block of 32 dims of a query has a size of its own, and some dims of it another; keys are as much smaller or
    larger, so that every block weighs alike.  (Products are those of normal pairs, and so is the bound.)"""

    batch = MxPaged(22, new, kv, bits=bits, dtype=dtype, dim=dim, heads=4, kv_heads=2)
    batch.hint = hint
    rng = np.random.default_rng([6, dim])
    size = np.zeros((2, dim))
    for g in range(2):
        size[g] = np.repeat(rng.permutation([-9, 0, 5, -3])[:dim // 32], 32)
        size[g] += np.where(rng.random(dim) < 0.1, rng.choice([-3, 4], dim), 0)
    batch.q = (batch.q.double() * 2.0**torch.from_numpy(np.repeat(size, 2, axis=0))).to(dtype)
    batch.k = (batch.k.double() * 2.0**-torch.from_numpy(size)[:, None, :]).to(dtype)
    batch.repack()
    _check(batch, native)


@each_form
def test_large_scores_in_heads_of_128(torch_gpu, native, dtype, bits, new, kv, hint):
    """Scores of up to a hundred and a first key that outweighs the others by far."""

    batch = MxPaged(23, new, kv, bits=bits, dtype=dtype, dim=128, heads=4, kv_heads=2)
    batch.hint = hint
    batch.k = batch.k.nan_to_num(0.0) * 12
    batch.v = batch.v.nan_to_num(0.0)
    page = batch.table[0, 0]
    batch.k[page, :, 0] = -batch.q[0, :2] * 8
    batch.repack()
    # sum |q k| * scale: 128 normal pairs with keys of 18 have 130, below 2^8 here; 128 * 2^-24 of that is 2^-9 of a
    # weight, and again of the weights' sum
    _check(batch, native, off=2.0**-8 + 2.0**-11)
