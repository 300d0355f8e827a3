"""GPU: attention over a paged cache with the kernel for few rows of long caches, against softmax in 64 bits.

The plan counts the told longest length up to a row of the page table, so a batch comes to this kernel, which
otherwise takes many long sequences, where both have room for 2^20 keys: the tests of the small batches, with such
tables.  Their rows of more than 16 a KV head, and what those share a batch with, go by the plan as ever."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import tests.test_gpu_paged_attention as small
from tests._paged_ref import Paged, f64

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16
ROOM = 1 << 20


class Roomy(Paged):
    def __init__(self, *args, **kwargs):
        super().__init__(*args, **kwargs)
        table = np.full((len(self.kv), ROOM // self.page), -7, dtype=np.int32)
        table[:, :self.table.shape[1]] = self.table
        self.table = table
        self.hint = ROOM


@pytest.fixture(autouse=True)
def roomy(monkeypatch):
    monkeypatch.setattr(small, "Paged", Roomy)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("new,kv,heads,kv_heads,page,layout", [
    # one key, the ends of units of 32 keys and of the waves' rounds of 128
    ([1], [1], 1, 1, 1, "hnd"),
    ([1, 1, 1, 1], [1, 31, 32, 33], 16, 2, 16, "hnd"),
    ([1, 1, 1], [127, 129, 1000], 7, 1, 16, "nhd"),
    ([1] * 9, [5, 700, 1, 64, 65, 333, 16, 17, 2000], 12, 4, 64, "hnd"),
    ([1, 1], [70, 3], 16, 1, 1, "nhd"),
    # drafts, up to 16 columns; no new tokens, no cache rows, rows that see no key
    ([3, 2, 4], [3, 100, 260], 8, 2, 16, "hnd"),
    ([16, 1, 5], [200, 0, 5], 2, 2, 16, "hnd"),
    ([0, 4, 0, 1, 3], [9, 4, 0, 0, 1], 4, 2, 16, "hnd"),
    # beside chunks
    ([33, 200, 1, 64], [33, 500, 77, 64], 8, 4, 16, "hnd"),
    ([250, 5], [1300, 5], 7, 7, 128, "nhd"),
    ([1, 130, 1], [900, 131, 2], 16, 2, 4096, "hnd"),
    # many sequences, a thread's run of them, and a long one in many stretches
    ([1] * 300, list(range(1, 301)), 4, 2, 16, "hnd"),
    ([1, 0, 2] * 100, [300, 4, 129] * 100, 2, 2, 64, "nhd"),
    ([4, 1], [40000, 9], 8, 2, 16, "hnd"),
])
def test_matches_fp64(torch_gpu, native, dtype, dim, new, kv, heads, kv_heads, page, layout):
    small.test_matches_fp64(torch_gpu, native, dtype, dim, new, kv, heads, kv_heads, page, layout, ROOM)


@pytest.mark.parametrize("new,kv", [([1, 1], [3000, 700]), ([60], [2500]), ([1, 90, 2], [4000, 1500, 1])])
def test_splits_follow_the_workspace_and_the_hints(torch_gpu, native, new, kv):
    batch = Roomy(5, new, kv, heads=8, kv_heads=2, dim=128)
    d = batch.device()
    nbytes = native.lib.kudacuda_paged_attention_workspace_bytes(batch.tokens, len(new), max(new), ROOM, 8, 2, 128)
    row = batch.tokens * 8 * 130 * 4
    for size in (0, row - 16, 2 * row, 3 * row + 16, 6 * row, nbytes):
        d["out"].fill_(7.25)
        small._check(batch, batch.call(native, d, nbytes=size))
    for max_new, max_kv in ((1, 1), (1, ROOM), (batch.tokens, 1), (1 << 20, 1 << 30)):
        d["out"].fill_(7.25)
        small._check(batch, batch.call(native, d, max_new=max_new, max_kv=max_kv))


@pytest.mark.parametrize("new,kv", [([1, 1, 1], [900, 33, 0]), ([70, 3], [200, 3])])
def test_rows_behind_the_last_sequence_stay(torch_gpu, native, new, kv):
    small.test_rows_behind_the_last_sequence_stay(torch_gpu, native, new, kv, ROOM)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("new,kv", [([4], [300]), ([150, 2], [400, 90])])
def test_infinities_and_nan_of_hidden_keys_stay_hidden(torch_gpu, native, dtype, new, kv):
    if len(kv) == 1:
        small.test_infinities_and_nan_of_hidden_keys_stay_hidden(torch_gpu, native, dtype, new, kv, ROOM)
        return
    batch = Roomy(8, new, kv, dtype=dtype, dim=64)
    page, at = batch.table[1, 89 // 16], 89 % 16
    batch.k[page, :, at] = batch.v[page, :, at] = float("nan")
    out = batch.call(native, batch.device())
    small._check(batch, out, rows=np.arange(151))
    assert np.isnan(f64(out[-1])).all()


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_large_scores_and_lowest_values(torch_gpu, native, dtype):
    small.test_large_scores_and_lowest_values(torch_gpu, native, dtype, ROOM)


def test_pages_outside_the_pool_make_nan_rows(torch_gpu, native):
    small.test_pages_outside_the_pool_make_nan_rows(torch_gpu, native, ROOM)


def test_lengths_that_do_not_fit_the_table_make_nan_rows(torch_gpu, native):
    for new, kv in (([1, 1], [64, 40]), ([50, 3], [64, 40]), ([3, 50], [64, 40])):
        for bad in (-1, ROOM + 1, 2**31 - 1):
            batch = Roomy(11, new, kv)
            d = batch.device()
            d["lens"][0] = bad
            for nbytes in (None, 0, 1 << 20):
                out = f64(batch.call(native, d, nbytes=nbytes))
                assert np.isnan(out[:new[0]]).all()
                small._check(batch, d["out"], rows=np.arange(new[0], batch.tokens))


def test_starts_outside_the_rows_stay_inside(torch_gpu, native):
    small.test_starts_outside_the_rows_stay_inside(torch_gpu, native, ROOM)


def test_starts_that_descend_stay_inside(torch_gpu, native):
    small.test_starts_that_descend_stay_inside(torch_gpu, native, ROOM)


def test_captured_call_follows_its_tables(torch_gpu, native):
    small.test_captured_call_follows_its_tables(torch_gpu, native, ROOM)


def test_results_do_not_change_from_call_to_call(torch_gpu, native):
    small.test_results_do_not_change_from_call_to_call(torch_gpu, native, ROOM)


@pytest.mark.parametrize("new,kv,heads", [
    ([1], [5000], 16), ([1] * 40, [900, 3, 64, 0, 2000] * 8, 8), ([3, 4, 1] * 20, [700, 30, 2500] * 20, 8),
    ([90, 1, 1], [1200, 7000, 40], 16)])
def test_calls_stay_inside_their_workspace(torch_gpu, native, new, kv, heads):
    small.test_calls_stay_inside_their_workspace(torch_gpu, native, new, kv, heads, ROOM)
