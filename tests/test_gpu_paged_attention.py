"""GPU: attention of new tokens over a paged cache (kudacuda_paged_attention) against softmax in 64 bits.

Rows of the pools that no sequence has hold NaN, table entries behind a sequence's pages no valid id."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from tests._paged_ref import Paged, f64

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16
# A told longest length of 2^20 puts sequences of few rows into the kernel for them, which otherwise takes large batches.
hints = pytest.mark.parametrize("hint", [None, 1 << 20])


def _check(batch, out, rows=None):
    want, size = batch.want()
    got = f64(out)
    rows = np.arange(int(batch.starts[-1])) if rows is None else rows
    off = np.abs(got[rows] - want[rows])
    assert np.isfinite(got[rows]).all()
    bound = batch.bound(want, size)[rows]
    assert (off <= bound).all(), float((off / np.maximum(bound, 1e-30)).max())


@hints
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("new,kv,heads,kv_heads,page,layout", [
    # single tokens: one key, the ends of units of 32 keys and of the waves' rounds of 128
    ([1], [1], 1, 1, 1, "hnd"),
    ([1, 1, 1, 1], [1, 31, 32, 33], 16, 2, 16, "hnd"),
    ([1, 1, 1], [127, 129, 1000], 7, 1, 16, "nhd"),
    ([1] * 9, [5, 700, 1, 64, 65, 333, 16, 17, 2000], 12, 4, 64, "hnd"),
    ([1, 1], [300, 40], 32, 1, 8, "nhd"),            # 32 heads of a KV head: past the few-row form
    ([1, 1], [70, 3], 64, 1, 16, "hnd"),
    # few new tokens: drafts, on both sides of 16 columns
    ([3, 2, 4], [3, 100, 260], 8, 2, 16, "hnd"),
    # chunks: first ones (no cache before), later ones, ends inside a tile and a window
    ([17], [17], 4, 2, 16, "hnd"),
    ([128], [128], 2, 2, 64, "nhd"),
    ([33, 200, 1, 64], [33, 500, 77, 64], 8, 4, 16, "hnd"),
    ([250, 5], [1300, 5], 7, 7, 128, "nhd"),
    ([1, 130, 1], [900, 131, 2], 16, 2, 4096, "hnd"),
    # sequences without new tokens, without cache rows, and rows that see no key
    ([0, 4, 0, 1, 40], [9, 4, 0, 0, 13], 4, 2, 16, "hnd"),
    ([2, 60], [0, 1], 4, 4, 16, "hnd"),
    # pages smaller than what a wave loads at once, in tiles
    ([90, 1, 33], [260, 7, 33], 4, 2, 1, "hnd"),
    ([150], [390], 2, 1, 2, "nhd"),
    # tiles enough for two blocks a CU, many sequences
    ([2048], [2100], 32, 32, 16, "hnd"),
    ([40, 0, 7, 100] * 70, [41, 5, 30, 100] * 70, 2, 2, 16, "hnd"),
    ([1] * 300, list(range(1, 301)), 4, 2, 16, "hnd"),
    # one tile a KV head: more than 64 splits, splits that even out lengths, with empty ones among them
    ([4], [40000], 16, 2, 16, "hnd"),
    ([1, 1], [30000, 31], 32, 1, 64, "nhd"),
    ([4, 0, 3, 4, 2] * 6, [3000, 5, 3, 1999, 64] * 6, 12, 2, 16, "hnd"),
    ([1] * 10, [2000, 1, 64, 65, 0, 1500, 3, 128, 127, 700], 32, 1, 16, "nhd"),
])
def test_matches_fp64(torch_gpu, native, dtype, dim, new, kv, heads, kv_heads, page, layout, hint):
    batch = Paged(len(new) + sum(kv), new, kv, heads=heads, kv_heads=kv_heads, dim=dim, page=page, dtype=dtype,
                  layout=layout, q_extra=1)
    batch.hint = hint
    print(f"paged attention {new} of {kv}, {heads}/{kv_heads} heads of {dim}, pages of {page}", flush=True)
    _check(batch, batch.call(native, batch.device()))


@pytest.mark.parametrize("new,kv", [([1, 1], [3000, 700]), ([60], [2500]), ([1, 90, 2], [4000, 1500, 1])])
def test_splits_follow_the_workspace_and_the_hints(torch_gpu, native, new, kv):
    """No workspace, a small one and a full one; hints that are too small and too large: the same results to rounding."""

    batch = Paged(5, new, kv, heads=8, kv_heads=2, dim=128)
    d = batch.device()
    nbytes = native.lib.kudacuda_paged_attention_workspace_bytes(batch.tokens, len(new), max(new), max(kv), 8, 2, 128)
    assert nbytes > 0
    row = batch.tokens * 8 * 130 * 4
    for size in (0, row - 16, 2 * row, 3 * row + 16, nbytes):
        d["out"].fill_(7.25)
        _check(batch, batch.call(native, d, nbytes=size))
    for max_new, max_kv in ((1, 1), (1, 1 << 20), (batch.tokens, 1), (1 << 20, 1 << 20)):
        d["out"].fill_(7.25)
        _check(batch, batch.call(native, d, max_new=max_new, max_kv=max_kv))


@hints
@pytest.mark.parametrize("new,kv", [([1, 1, 1], [900, 33, 0]), ([70, 3], [200, 3])])
def test_rows_behind_the_last_sequence_stay(torch_gpu, native, new, kv, hint):
    batch = Paged(6, new, kv, extra_rows=5)
    batch.hint = hint
    for nbytes in (None, 0):
        d = batch.device()
        out = batch.call(native, d, nbytes=nbytes)
        _check(batch, out)
        assert (f64(out[-5:]) == 7.25).all()


@hints
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("new,kv", [([4], [300]), ([150], [400])])
def test_infinities_and_nan_of_hidden_keys_stay_hidden(torch_gpu, native, dtype, new, kv, hint):
    """The last key's K and V are NaN and infinite: only the row that sees it is not finite."""

    batch = Paged(8, new, kv, dtype=dtype, dim=64)
    batch.hint = hint
    last = kv[0] - 1
    page, at = batch.table[0, last // 16], last % 16
    for value in (float("inf"), float("nan")):
        batch.k[page, :, at] = value if value != value else 3.0
        batch.v[page, :, at] = value
        d = batch.device()
        for nbytes in (None, 0):
            out = batch.call(native, d, nbytes=nbytes)
            _check(batch, out, rows=np.arange(new[0] - 1))
            assert not np.isfinite(f64(out[-1])).any()


@hints
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_large_scores_and_lowest_values(torch_gpu, native, dtype, hint):
    """Scores of hundreds, keys at the type's lowest value, a first key that outweighs all others by far."""

    batch = Paged(9, [1, 40], [600, 300], dtype=dtype, dim=64, junk=float("-inf"))
    batch.hint = hint
    batch.k *= 12
    page = batch.table[0, 0]
    batch.k[page, :, 3] = 0
    batch.v[page, :, 3] = torch.finfo(dtype).min / 4
    batch.k[page, :, 4] = -batch.q[0, :2] * 8
    want, size = batch.want()
    out = f64(batch.call(native, batch.device()))
    assert np.isfinite(out).all()
    # scores of up to 64 * 12 * 4 * 1.5 / 8: 2^10 of them in fp32, off by 64 * 2^-24 * 2^10 = 2^-8
    bound = batch.bound(want, size) + 2.0**-7 * size
    assert (np.abs(out - want) <= bound).all()


@hints
def test_pages_outside_the_pool_make_nan_rows(torch_gpu, native, hint):
    """A bad page id is not read; the rows that see one of its keys are NaN, the others hold."""

    for new, kv in (([1, 1, 1], [500, 90, 33]), ([40, 1], [300, 20])):
        for bad in (-1, 2**31 - 1, None):
            batch = Paged(10, new, kv)
            batch.hint = hint
            d = batch.device()
            d["table"][0, (kv[0] - 1) // 16 - 1] = batch.num_pages if bad is None else bad
            first = ((kv[0] - 1) // 16 - 1) * 16  # the first key of that page
            for nbytes in (None, 0):
                out = f64(batch.call(native, d, nbytes=nbytes))
                for i in range(new[0]):
                    seen = kv[0] - new[0] + i >= first
                    assert np.isnan(out[i]).all() if seen else np.isfinite(out[i]).all(), (new, bad, i)
                _check(batch, d["out"], rows=np.array([i for i in range(batch.tokens) if np.isfinite(out[i]).all()]))
                assert np.isfinite(out[new[0]:]).all()


@hints
def test_lengths_that_do_not_fit_the_table_make_nan_rows(torch_gpu, native, hint):
    for new, kv in (([1, 1], [64, 40]), ([50, 3], [64, 40])):
        for bad in (-1, 4 * 16 + 1, 2**31 - 1):
            batch = Paged(11, new, kv)
            batch.hint = hint
            d = batch.device()
            d["lens"][0] = bad
            for nbytes in (None, 0, 1 << 20):
                out = f64(batch.call(native, d, nbytes=nbytes))
                assert np.isnan(out[:new[0]]).all()
                _check(batch, d["out"], rows=np.arange(new[0], batch.tokens))


@hints
def test_starts_outside_the_rows_stay_inside(torch_gpu, native, hint):
    """Starts past the tokens (and below zero) name no rows."""

    batch = Paged(12, [2, 3], [40, 50])
    batch.hint = hint
    d = batch.device()
    d["starts"].copy_(torch.tensor([-4, 2, 2**31 - 1], dtype=torch.int32))
    out = f64(batch.call(native, d, nbytes=0))
    assert np.isfinite(out).all()


@hints
def test_offsets_past_32_bits(torch_gpu, native, hint):
    """Pools of more than 2^32 elements: pages 2^25 elements apart, the values half a page behind the keys."""

    stride, pages = 1 << 25, 130
    batch = Paged(13, [1, 20], [700, 300], dim=64, kv_heads=2, heads=4, spare=pages - 3 - 44 - 19)
    batch.hint = hint
    assert batch.num_pages == pages and int(batch.table.max()) > 127
    d = batch.device()
    pool = torch.zeros(pages * stride, dtype=BF16, device="cuda:0")
    shape, inner = (pages, 2, 16, 64), (2 * 16 * 64) // 2
    k = torch.as_strided(pool, shape, (stride, inner, 64, 1), 0)
    v = torch.as_strided(pool, shape, (stride, inner, 64, 1), stride // 2)
    k.copy_(d["k"])
    v.copy_(d["v"])
    d |= {"k": k, "v": v, "strides": (stride, inner, 64)}
    _check(batch, batch.call(native, d))
    del pool, k, v, d
    torch.cuda.empty_cache()


def test_two_streams_and_a_second_handle(torch_gpu, native):
    from kudacuda_amd._native import Native

    other = Native(0)
    first, second = Paged(14, [1, 1], [2000, 900], dim=128), Paged(15, [100], [800], dim=128)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    ds = [first.device(), second.device()]
    torch.cuda.synchronize()
    for _ in range(5):
        first.call(native, ds[0], stream=streams[0])
        second.call(native, ds[1], stream=streams[1])
        second.call(other, ds[1], stream=streams[1])
    torch.cuda.synchronize()
    _check(first, ds[0]["out"])
    _check(second, ds[1]["out"])
    other.close()


@hints
def test_captured_call_follows_its_tables(torch_gpu, native, hint):
    """One capture, replayed while the sequences grow: lengths, tables and starts are read at replay time."""

    batch = Paged(16, [1, 1, 1], [900, 600, 40], dim=128)
    d = batch.device()
    nbytes = native.lib.kudacuda_paged_attention_workspace_bytes(3, 3, 1, hint or 1024, 4, 2, 128)
    workspace = torch.zeros(nbytes, dtype=torch.uint8, device="cuda:0")
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        batch.call(native, d, stream=torch.cuda.current_stream(), workspace=workspace, nbytes=nbytes, max_kv=hint or 1024)
    for kv in ([900, 600, 40], [1, 600, 39], [33, 0, 17], [899, 128, 40]):
        batch.kv = kv
        with torch.cuda.stream(side):
            d["lens"].copy_(torch.tensor(kv, dtype=torch.int32))
            d["out"].fill_(7.25)
            graph.replay()
        side.synchronize()
        _check(batch, d["out"])
        replayed = d["out"].clone()
        batch.call(native, d, workspace=workspace, nbytes=nbytes, max_kv=hint or 1024)
        torch.cuda.synchronize()
        assert torch.equal(replayed, d["out"])


@hints
def test_results_do_not_change_from_call_to_call(torch_gpu, native, hint):
    batch = Paged(17, [1, 200, 3], [3000, 900, 60], dim=128, heads=16)
    batch.hint = hint
    d = batch.device()
    first = batch.call(native, d).clone()
    for _ in range(5):
        assert torch.equal(batch.call(native, d), first)


@hints
def test_starts_that_descend_stay_inside(torch_gpu, native, hint):
    """Starts that go back and forth name no batch: whatever the rows become, the sequences' pages and the workspace
    hold what they held, and the next call is right."""

    for new, kv in (([1] * 6, [400, 30, 70, 2000, 5, 90]), ([70, 1, 40, 3], [300, 20, 100, 50])):
        batch = Paged(18, new, kv, dim=128)
        batch.hint = hint
        d = batch.device()
        nbytes = native.lib.kudacuda_paged_attention_workspace_bytes(batch.tokens, len(new), max(new), hint or max(kv),
                                                                          4, 2, 128)
        workspace = torch.full((nbytes + 4096,), 0x7f, dtype=torch.uint8, device="cuda:0")
        pools = d["k"].clone(), d["v"].clone()
        good = d["starts"].clone()
        d["starts"].copy_(torch.tensor([0, batch.tokens] * 4, dtype=torch.int32)[:len(new) + 1])
        batch.call(native, d, workspace=workspace, nbytes=nbytes)
        torch.cuda.synchronize()
        assert (workspace[nbytes:] == 0x7f).all()
        assert all(torch.equal(a.view(torch.int16), b.view(torch.int16)) for a, b in zip(pools, (d["k"], d["v"])))
        d["starts"].copy_(good)
        _check(batch, batch.call(native, d, workspace=workspace, nbytes=nbytes))


def test_cache_calls_captured_twice_do_not_share_a_workspace(torch_gpu, native):
    """Two graphs with attention over many splits, replayed at the same time on two streams."""

    from kudacuda_amd.paged_cache import PagedKvCache

    cache = PagedKvCache(native, torch, layers=1, kv_heads=2, head_dim=128, num_pages=400, page_size=16)
    cache.pool.normal_()
    batches = []
    for n in (3000, 2500):
        s = cache.create()
        cache.extend([s], [n])
        batches.append(cache.extend([s], [1]))
    q = torch.randn((2, 1, 16, 128), device="cuda:0").bfloat16()
    want = [cache.attend(0, b, x).clone() for b, x in zip(batches, q)]
    outs = [torch.zeros_like(w) for w in want]
    torch.cuda.synchronize()
    graphs, streams = [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for b, x, out, s in zip(batches, q, outs, streams):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=s):
            cache.attend(0, b, x, out=out)
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        for s in streams:
            s.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))
        assert torch.equal(cache.attend(0, batches[0], q[0]), want[0])
        torch.cuda.synchronize()


@hints
@pytest.mark.parametrize("new,kv,heads", [
    ([1], [5000], 16), ([1] * 40, [900, 3, 64, 0, 2000] * 8, 8), ([3, 4, 1] * 20, [700, 30, 2500] * 20, 8), ([700], [900], 4),
    ([90, 1, 1], [1200, 7000, 40], 16)])
def test_calls_stay_inside_their_workspace(torch_gpu, native, new, kv, heads, hint):
    """Of the told size and of less."""

    batch = Paged(19, new, kv, heads=heads, dim=128)
    batch.hint = hint
    d = batch.device()
    full = native.lib.kudacuda_paged_attention_workspace_bytes(batch.tokens, len(new), max(new), hint or max(kv), heads, 2, 128)
    for nbytes in (full, full // 2 // 16 * 16, full // 5 // 16 * 16):
        workspace = torch.full((nbytes + 4096,), 0x7f, dtype=torch.uint8, device="cuda:0")
        _check(batch, batch.call(native, d, workspace=workspace, nbytes=nbytes))
        assert (workspace[nbytes:] == 0x7f).all()
