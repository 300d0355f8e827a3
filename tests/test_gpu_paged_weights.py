"""GPU: what attention over a paged cache does with single weights: small ones beside a large one, their rounding,
and that no key of a long cache is left out.  Against softmax in 64 bits."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from tests._paged_ref import f64
from tests._paged_weights import marked, one_above_a_tail, opposite_roundings, told, weight_bound

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16
# (a longest length of 2^20, where the table has room for it, takes the kernel for few rows of long caches)
hints = pytest.mark.parametrize("hint", [None, 1 << 20])


def _check(native, batch, hint):
    told(batch, hint)
    want, size = batch.want()
    bound = weight_bound(batch, want, size)
    d = batch.device()
    for nbytes in (None, 0):  # the keys split over the chip, and in one piece
        d["out"].fill_(7.25)
        off = np.abs(f64(batch.call(native, d, nbytes=nbytes)) - want)
        assert (off <= bound).all(), (nbytes, float((off / np.maximum(bound, 1e-30)).max()))


@hints
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("new", [[1], [40]])
@pytest.mark.parametrize("gap", [16.0, 20.0, 24.5, 25.0, 28.25])
def test_a_long_tail_beside_one_large_weight_counts(torch_gpu, native, dtype, dim, new, gap, hint):
    for key in (5, 20011, 39950):
        print(f"tail of 40000 keys 2^-{gap} below key {key}, {new} new", flush=True)
        _check(native, one_above_a_tail(new, [40000], key, gap, heads=4, kv_heads=2, dim=dim, dtype=dtype), hint)


@hints
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("new,kv,heads,kv_heads", [
    ([1], [500], 16, 2), ([1], [2000], 16, 2), ([4], [900], 16, 2), ([2], [777], 32, 2), ([1], [300], 32, 1),
    ([1] * 20, [200, 33, 1999, 64] * 5, 16, 2), ([100, 1, 3], [400, 900, 130], 16, 2), ([33], [500], 2, 2)])
def test_weights_of_few_rows_keep_two_parts(torch_gpu, native, dtype, dim, new, kv, heads, kv_heads, hint):
    print(f"weights of {new} of {kv}, {heads}/{kv_heads} heads of {dim}", flush=True)
    _check(native, opposite_roundings(new, kv, heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype), hint)


@hints
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("edges", [False, True])
@pytest.mark.parametrize("new,kv,heads,kv_heads", [
    ([1], [40000], 16, 2), ([4], [40000], 16, 2), ([40], [40000], 4, 2), ([600], [9000], 4, 2),
    ([1, 200], [9999, 5000], 8, 2)])
def test_every_window_of_a_long_cache_counts(torch_gpu, native, dtype, dim, edges, new, kv, heads, kv_heads, hint):
    print(f"marked windows, {new} of {kv}, {heads}/{kv_heads} heads of {dim}", flush=True)
    _check(native, marked(new, kv, edges, heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype), hint)
