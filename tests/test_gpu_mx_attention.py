"""GPU: attention over a cache of 8 or 4 bits against softmax in 64 bits on the numbers that its pages hold.

Rows that no sequence has hold NaN blocks, table entries behind a sequence's pages no valid id.  The sums are those of
the attention over 16-bit pages, and so are the bounds."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from kudacuda_amd.paged_cache import PagedKvCache
from tests._mx_ref import BLOCK, MxPaged, page_bytes
from tests._paged_ref import f64

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16
# A told longest length of 2^20 puts sequences of few rows into the kernel for them, which otherwise takes large batches.
hints = pytest.mark.parametrize("hint", [None, 1 << 20])
all_bits = pytest.mark.parametrize("bits", [4, 8])


def _check(batch, out, rows=None):
    want, size = batch.want()
    got = f64(out)
    rows = np.arange(int(batch.starts[-1])) if rows is None else rows
    off = np.abs(got[rows] - want[rows])
    assert np.isfinite(got[rows]).all()
    bound = batch.bound(want, size)[rows]
    assert (off <= bound).all(), float((off / np.maximum(bound, 1e-30)).max())


@hints
@all_bits
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("new,kv,heads,kv_heads,page", [
    # single tokens: one key, the ends of units of 16, 32 and 64 keys and of the waves' rounds
    ([1], [1], 1, 1, 16),
    ([1, 1, 1, 1, 1], [1, 31, 32, 33, 17], 16, 2, 16),
    ([1, 1, 1, 1], [127, 129, 1000, 256], 7, 1, 64),
    ([1] * 9, [5, 700, 1, 64, 65, 333, 16, 17, 2000], 12, 4, 64),
    ([1, 1], [300, 40], 32, 1, 16),            # 32 heads of a KV head: past the few-row form
    ([1, 1], [70, 3], 64, 1, 16),
    # few new tokens: drafts, on both sides of 16 columns
    ([3, 2, 4], [3, 100, 260], 8, 2, 16),
    # chunks: first ones (no cache before), later ones, ends inside a tile and a window
    ([17], [17], 4, 2, 16),
    ([128], [128], 2, 2, 64),
    ([33, 200, 1, 64], [33, 500, 77, 64], 8, 4, 16),
    ([250, 5], [1300, 5], 7, 7, 128),
    ([1, 130, 1], [900, 131, 2], 16, 2, 4096),
    # chunks behind a past as long and longer, tiles enough for blocks of one K-group and splits
    ([300, 1, 200, 64, 130], [2700, 900, 3000, 64, 131], 24, 12, 16),
    # sequences without new tokens, without cache rows, and rows that see no key
    ([0, 4, 0, 1, 40], [9, 4, 0, 0, 13], 4, 2, 16),
    ([2, 60], [0, 1], 4, 4, 16),
    # tiles enough for two blocks a CU, many sequences
    ([2048], [2100], 32, 32, 16),
    ([40, 0, 7, 100] * 70, [41, 5, 30, 100] * 70, 2, 2, 16),
    ([1] * 300, list(range(1, 301)), 4, 2, 16),
    # as many sequences as a wave has lanes, and one more
    ([1, 2, 0, 1] * 16, [(i * 37) % 900 for i in range(64)], 8, 2, 16),
    ([1, 2, 0, 1] * 16 + [3], [(i * 37) % 900 for i in range(64)] + [1500], 8, 2, 16),
    # one tile a KV head: more than 64 splits, splits that even out lengths, with empty ones among them
    ([4], [20000], 16, 2, 16),
    ([1, 1], [30000, 31], 32, 1, 64),
    ([4, 0, 3, 4, 2] * 6, [3000, 5, 3, 1999, 64] * 6, 12, 2, 16),
    ([1] * 10, [2000, 1, 64, 65, 0, 1500, 3, 128, 127, 700], 32, 1, 16),
])
def test_matches_fp64(torch_gpu, native, dtype, bits, dim, new, kv, heads, kv_heads, page, hint):
    batch = MxPaged(len(new) + sum(kv), new, kv, bits=bits, heads=heads, kv_heads=kv_heads, dim=dim, page=page, dtype=dtype,
                    q_extra=1, extra=16 * (len(new) % 3))
    batch.hint = hint
    print(f"attention in {bits} bits, {new[:9]} of {kv[:9]}, {heads}/{kv_heads} heads of {dim}, pages of {page}", flush=True)
    _check(batch, batch.call(native, batch.device()))


@all_bits
@pytest.mark.parametrize("new,kv", [([1, 1], [3000, 700]), ([60], [2500]), ([1, 90, 2], [4000, 1500, 1])])
def test_splits_follow_the_workspace_and_the_hints(torch_gpu, native, bits, new, kv):
    """No workspace, a small one and a full one; hints that are too small and too large: the same results to rounding."""

    batch = MxPaged(5, new, kv, bits=bits, heads=8, kv_heads=2, dim=128)
    d = batch.device()
    nbytes = batch.workspace_bytes(native)
    assert nbytes > 0
    row = batch.tokens * 8 * 130 * 4
    for size in (0, row - 16, 2 * row, 3 * row + 16, nbytes):
        d["out"].fill_(7.25)
        _check(batch, batch.call(native, d, nbytes=size))
    for max_new, max_kv in ((1, 1), (1, 1 << 20), (batch.tokens, 1), (1 << 20, 1 << 20)):
        d["out"].fill_(7.25)
        _check(batch, batch.call(native, d, max_new=max_new, max_kv=max_kv))


@hints
@all_bits
@pytest.mark.parametrize("new,kv", [([1, 1, 1], [900, 33, 0]), ([70, 3], [200, 3])])
def test_rows_behind_the_last_sequence_stay(torch_gpu, native, bits, new, kv, hint):
    batch = MxPaged(6, new, kv, bits=bits, extra_rows=5)
    batch.hint = hint
    for nbytes in (None, 0):
        d = batch.device()
        out = batch.call(native, d, nbytes=nbytes)
        _check(batch, out)
        assert (f64(out[-5:]) == 7.25).all()


@hints
@all_bits
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("new,kv", [([4], [300]), ([150], [400])])
def test_nan_blocks_of_hidden_keys_stay_hidden(torch_gpu, native, dtype, bits, dim, new, kv, hint):
    """The last key's K or V has a NaN block: only the row that sees it is not finite, and of it only that block's dims
    where it is V's."""

    last = kv[0] - 1
    for of_keys in (True, False):
        batch = MxPaged(8, new, kv, bits=bits, dtype=dtype, dim=dim)
        batch.hint = hint
        (batch.k if of_keys else batch.v)[batch.table[0, last // 16], :, last % 16, dim - BLOCK] = float("nan")
        batch.repack()
        d = batch.device()
        for nbytes in (None, 0):
            out = batch.call(native, d, nbytes=nbytes)
            _check(batch, out, rows=np.arange(new[0] - 1))
            got = f64(out[new[0] - 1])
            assert np.isnan(got[:, dim - BLOCK:]).all()
            assert np.isnan(got).all() if of_keys else np.isfinite(got[:, :dim - BLOCK]).all()


@hints
@all_bits
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_large_scores_and_far_values(torch_gpu, native, bits, dtype, hint):
    """Scores of hundreds, a first key that outweighs all others by far, values of the type's upper range."""

    batch = MxPaged(9, [1, 40], [600, 300], bits=bits, dtype=dtype, dim=64)
    batch.hint = hint
    batch.k = batch.k.nan_to_num(0.0) * 12
    batch.v = batch.v.nan_to_num(0.0)
    page = batch.table[0, 0]
    batch.k[page, :, 3] = 0
    batch.v[page, :, 3] = torch.finfo(dtype).min / 4
    batch.k[page, :, 4] = -batch.q[0, :2] * 8
    batch.repack()
    want, size = batch.want()
    out = f64(batch.call(native, batch.device()))
    assert np.isfinite(out).all()
    # scores of up to 64 * 12 * 4 * 1.5 / 8: 2^10 of them in fp32, off by 64 * 2^-24 * 2^10 = 2^-8
    bound = batch.bound(want, size) + 2.0**-7 * size
    assert (np.abs(out - want) <= bound).all()


@hints
@all_bits
def test_pages_outside_the_pool_make_nan_rows(torch_gpu, native, bits, hint):
    """A bad page id is not read; the rows that see one of its keys are NaN, the others hold."""

    for new, kv in (([1, 1, 1], [500, 90, 33]), ([40, 1], [300, 20])):
        for bad in (-1, 2**31 - 1, None):
            batch = MxPaged(10, new, kv, bits=bits)
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
@all_bits
def test_lengths_that_do_not_fit_the_table_make_nan_rows(torch_gpu, native, bits, hint):
    for new, kv in (([1, 1], [64, 40]), ([50, 3], [64, 40])):
        for bad in (-1, 4 * 16 + 1, 2**31 - 1):
            batch = MxPaged(11, new, kv, bits=bits)
            batch.hint = hint
            d = batch.device()
            d["lens"][0] = bad
            for nbytes in (None, 0, 1 << 20):
                out = f64(batch.call(native, d, nbytes=nbytes))
                assert np.isnan(out[:new[0]]).all()
                _check(batch, d["out"], rows=np.arange(new[0], batch.tokens))


@hints
@all_bits
def test_offsets_past_32_bits(torch_gpu, native, bits, hint):
    """Pools of more than 2^32 bytes: pages 2^26 apart, the values half a page behind the keys."""

    stride, pages = 1 << 26, 130
    batch = MxPaged(13, [1, 20], [700, 300], bits=bits, dim=64, spare=pages - 3 - 44 - 19)
    batch.hint = hint
    assert batch.num_pages == pages and int(batch.table.max()) > 127
    d = batch.device()
    pool = torch.zeros(pages * stride, dtype=torch.uint8, device="cuda:0")
    k, v = (torch.as_strided(pool, tuple(d["k"].shape), (stride, 1), at) for at in (0, stride // 2))
    k.copy_(d["k"])
    v.copy_(d["v"])
    d |= {"k": k, "v": v, "stride": stride}
    _check(batch, batch.call(native, d))
    del pool, k, v, d
    torch.cuda.empty_cache()


def test_two_streams_and_a_second_handle(torch_gpu, native):
    from kudacuda_amd._native import Native

    other = Native(0)
    first, second = MxPaged(14, [1, 1], [2000, 900], bits=4, dim=128), MxPaged(15, [100], [800], bits=8, dim=128)
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
@all_bits
def test_captured_call_follows_its_tables(torch_gpu, native, bits, hint):
    """One capture, replayed while the sequences grow: lengths, tables and starts are read at replay time."""

    batch = MxPaged(16, [1, 1, 1], [900, 600, 40], bits=bits, dim=128)
    d = batch.device()
    nbytes = batch.workspace_bytes(native, 1, hint or 1024)
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
@all_bits
def test_results_do_not_change_from_call_to_call(torch_gpu, native, bits, hint):
    batch = MxPaged(17, [1, 200, 3], [3000, 900, 60], bits=bits, dim=128, heads=16)
    batch.hint = hint
    d = batch.device()
    first = batch.call(native, d).clone()
    for _ in range(5):
        assert torch.equal(batch.call(native, d), first)


@hints
@all_bits
def test_starts_that_descend_or_leave_the_rows_stay_inside(torch_gpu, native, bits, hint):
    for new, kv in (([1] * 6, [400, 30, 70, 2000, 5, 90]), ([70, 1, 40, 3], [300, 20, 100, 50])):
        batch = MxPaged(18, new, kv, bits=bits, dim=128)
        batch.hint = hint
        d = batch.device()
        nbytes = batch.workspace_bytes(native)
        workspace = torch.full((nbytes + 4096,), 0x7f, dtype=torch.uint8, device="cuda:0")
        pools = d["k"].clone(), d["v"].clone()
        good = d["starts"].clone()
        for starts in ([0, batch.tokens] * 4, [-4, 2] + [2**31 - 1] * 6):
            d["starts"].copy_(torch.tensor(starts, dtype=torch.int32)[:len(new) + 1])
            batch.call(native, d, workspace=workspace, nbytes=nbytes)
            torch.cuda.synchronize()
            assert (workspace[nbytes:] == 0x7f).all()
            assert torch.equal(pools[0], d["k"]) and torch.equal(pools[1], d["v"])
        d["starts"].copy_(good)
        _check(batch, batch.call(native, d, workspace=workspace, nbytes=nbytes))


@hints
@all_bits
@pytest.mark.parametrize("new,kv,heads", [
    ([1], [5000], 16), ([1] * 40, [900, 3, 64, 0, 2000] * 8, 8), ([3, 4, 1] * 20, [700, 30, 2500] * 20, 8), ([700], [900], 4),
    ([90, 1, 1], [1200, 7000, 40], 16)])
def test_calls_stay_inside_their_workspace(torch_gpu, native, bits, new, kv, heads, hint):
    """Of the told size and of less."""

    batch = MxPaged(19, new, kv, bits=bits, heads=heads, dim=128)
    batch.hint = hint
    d = batch.device()
    full = batch.workspace_bytes(native)
    for nbytes in (full, full // 2 // 16 * 16, full // 5 // 16 * 16):
        workspace = torch.full((nbytes + 4096,), 0x7f, dtype=torch.uint8, device="cuda:0")
        _check(batch, batch.call(native, d, workspace=workspace, nbytes=nbytes))
        assert (workspace[nbytes:] == 0x7f).all()


@all_bits
def test_cache_calls_captured_twice_do_not_share_a_workspace(torch_gpu, native, bits):
    """Two graphs with append and attention over many splits, replayed at the same time on two streams."""

    cache = PagedKvCache(native, torch, layers=1, kv_heads=2, head_dim=128, num_pages=400, page_size=16, bits=bits)
    freq = torch.zeros(64, dtype=torch.float64, device="cuda:0")
    batches, news = [], []
    for n in (3000, 2500):
        s = cache.create()
        k, v = (torch.randn((n, 2, 128), device="cuda:0").bfloat16() for _ in range(2))
        cache.append(0, cache.extend([s], [n]), torch.zeros((n, 16, 128), dtype=BF16, device="cuda:0"), k, v, freq)
        batches.append(cache.extend([s], [1]))
        news.append([torch.randn((1, h, 128), device="cuda:0").bfloat16() for h in (16, 2, 2)])
    assert cache.pool.shape[2] == page_bytes(2, 16, 128, bits)

    def step(batch, x, out):
        return cache.attend(0, batch, cache.append(0, batch, *x, freq), out=out)

    want = [step(b, x, None).clone() for b, x in zip(batches, news)]
    outs = [torch.zeros_like(w) for w in want]
    torch.cuda.synchronize()
    graphs, streams = [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for b, x, out, s in zip(batches, news, outs, streams):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=s):
            step(b, x, out)
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        for s in streams:
            s.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))
        assert torch.equal(step(batches[0], news[0], None), want[0])
        torch.cuda.synchronize()


@hints
@all_bits
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("new,kv", [([1, 1, 1], [40, 300, 7]), ([3, 1], [200, 50]), ([20, 15], [90, 15])])
def test_queries_without_a_number_spoil_their_own_rows_only(torch_gpu, native, dtype, bits, dim, new, kv, hint):
    """A query with a NaN, or with an infinity at a dim where its keys are positive: NaN rows, and no others."""

    batch = MxPaged(3, new, kv, bits=bits, heads=4, kv_heads=2, dim=dim, dtype=dtype)
    batch.hint = hint
    batch.k[..., dim - 1] = batch.k[..., dim - 1].abs() + 1.0
    batch.repack()
    want, size = batch.want()
    spoilt = np.zeros((batch.tokens, 4), dtype=bool)
    for row, head, d, value in ((0, 1, 0, "nan"), (1, 3, dim - 1, "inf"), (batch.tokens - 1, 0, dim - 1, "inf")):
        batch.q[row, head, d] = float(value)
        spoilt[row, head] = True
    got = f64(batch.call(native, batch.device()))
    assert np.isnan(got[spoilt]).all()
    assert (np.abs(got - want) <= batch.bound(want, size))[~spoilt].all()
