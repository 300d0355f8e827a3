"""GPU: page copies (kudacuda_copy_pages), refusals of the paged-cache entry points, and the cache that keeps the books."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from tests import _refusals

pytestmark = pytest.mark.gpu


def _copy(native, pool, pairs, pools, pages, size, page_stride, pool_stride, stream=None):
    table = np.ascontiguousarray(pairs, dtype=np.int32).reshape(-1, 2)
    stream = torch.cuda.current_stream() if stream is None else stream
    native.call("kudacuda_copy_pages", pool.data_ptr(), table.ctypes.data, len(table), pools, pages, size, page_stride,
                pool_stride, stream.cuda_stream)


@pytest.mark.parametrize("pools,pages,size,moves,gap,layout", [
    (1, 2, 16, 1, 0, "pools"),
    (3, 9, 4096 + 16, 4, 48, "pools"),
    (72, 30, 8192, 15, 0, "pools"),
    (2, 12, 16384 * 2 + 32, 6, 0, "pages"),   # a page's pools side by side
    (2, 2000, 64, 1000, 0, "pools"),          # more pairs than one launch takes
    (2, 1200, 16, 448, 16, "pages"),
])
def test_copies_are_exact_and_touch_nothing_else(torch_gpu, native, pools, pages, size, moves, gap, layout):
    rng = np.random.default_rng([size, moves])
    inner = size + gap
    page_stride, pool_stride = (inner, inner * pages) if layout == "pools" else (inner * pools, inner)
    data = rng.integers(0, 256, pools * pages * inner, dtype=np.uint8)
    pool = torch.from_numpy(data.copy()).cuda()
    order = rng.permutation(pages)
    pairs = np.stack([rng.choice(order[moves:], moves), order[:moves]], axis=1)  # a source may serve several
    pairs[-1, 0] = pairs[-1, 1]  # and a page may stay where it is
    _copy(native, pool, pairs, pools, pages, size, page_stride, pool_stride)
    want = data.copy()
    for i in range(pools):
        for a, b in pairs:
            at, to = i * pool_stride + a * page_stride, i * pool_stride + b * page_stride
            want[to:to + size] = data[at:at + size]
    assert np.array_equal(pool.cpu().numpy(), want)


def test_no_pairs_is_a_call_that_does_nothing(torch_gpu, native):
    pool = torch.arange(64, dtype=torch.uint8, device="cuda:0")
    native.call("kudacuda_copy_pages", pool.data_ptr(), 0, 0, 1, 4, 16, 16, 0, torch.cuda.current_stream().cuda_stream)
    _copy(native, pool, [(2, 2)], 1, 4, 16, 16, 0)
    assert torch.equal(pool.cpu(), torch.arange(64, dtype=torch.uint8))


def test_the_list_may_change_as_soon_as_the_call_returns(torch_gpu, native):
    """Eager and captured calls keep their own pairs."""

    pool = torch.arange(6 * 64, device="cuda:0").to(torch.int16).reshape(6, 64)
    clean = pool.clone()
    pairs = np.array([[0, 5]], dtype=np.int32)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        _copy(native, pool, pairs, 1, 6, 128, 128, 0, stream=torch.cuda.current_stream())
    pairs[:] = 1
    for _ in range(3):
        pool.copy_(clean)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graph.replay()
        side.synchronize()
        assert torch.equal(pool[5], clean[0]) and torch.equal(pool[:5], clean[:5])


@pytest.mark.parametrize("name", list(_refusals.CALLS))
def test_refusals_leave_a_reason(torch_gpu, native, name):
    buffer = torch.zeros(1 << 22, dtype=torch.uint8, device="cuda:0")
    lib = native.lib
    stand_in = range(_refusals.P, _refusals.Q + 16)
    for call, args, reason in _refusals.refusals():
        if call == name:
            args = [buffer.data_ptr() + a - _refusals.P if a in stand_in else a for a in args]
            status = getattr(lib, call)(native.handle, *args)
            assert status == 1 and reason in native.error(), (call, args, native.error())
    torch.cuda.synchronize()
    assert int(buffer.count_nonzero()) == 0


def _cache(native, **kw):
    from kudacuda_amd.paged_cache import PagedKvCache

    kw = dict(layers=2, kv_heads=2, head_dim=64, num_pages=24, page_size=8) | kw
    return PagedKvCache(native, torch, **kw)


def _fill(cache, batch, rng, truth):
    """Random rows for a batch's tokens into every layer, and into ``truth`` {sequence: [layers][keys, values] rows}."""

    freq = torch.from_numpy(np.zeros(cache.head_dim // 2)).cuda()  # no turn: rows are stored as they are
    starts = batch.query_starts.cpu().numpy()
    for layer in range(cache.layers):
        k, v = (torch.from_numpy(rng.standard_normal((batch.tokens, cache.kv_heads, cache.head_dim)).astype(np.float32))
                .to(cache.pool.dtype).cuda() for _ in range(2))
        q = torch.zeros((batch.tokens, 4, cache.head_dim), dtype=cache.pool.dtype, device="cuda:0")
        cache.append(layer, batch, q, k, v, freq)
        for i, s in enumerate(batch.sequences):
            rows = truth.setdefault(s, [[[], []] for _ in range(cache.layers)])[layer]
            rows[0] += list(k[starts[i]:starts[i + 1]].cpu())
            rows[1] += list(v[starts[i]:starts[i + 1]].cpu())


def _holds(cache, truth):
    for s, layers in truth.items():
        pages, n = cache.pages(s), cache.length(s)
        for layer, rows in enumerate(layers):
            for pool, want in zip((cache.keys(layer), cache.values(layer)), rows):
                got = pool[pages].transpose(1, 2).flatten(0, 1)[:n].cpu()
                assert torch.equal(got, torch.stack(want)), (s, layer)


def test_forks_share_until_they_write_and_compaction_keeps_every_row(torch_gpu, native):
    cache, rng, truth = _cache(native), np.random.default_rng(4), {}
    a, b = cache.create(), cache.create()
    _fill(cache, cache.extend([a, b], [13, 8]), rng, truth)
    c, d = cache.fork(a), cache.fork(a)
    for s in (c, d):
        truth[s] = [[list(r) for r in layer] for layer in truth[a]]
    assert cache.pages(c) == cache.pages(a) and cache.free_pages == 24 - 3
    _fill(cache, cache.extend([a, c, d], [1, 2, 4]), rng, truth)  # all three write into the shared page at once
    assert len({cache.pages(s)[1] for s in (a, c, d)}) == 3 and len({cache.pages(s)[0] for s in (a, c, d)}) == 1
    _holds(cache, truth)
    _fill(cache, cache.extend([b], [30]), rng, truth)
    cache.free(a)
    truth.pop(a)
    cache.truncate(b, 17)
    truth[b] = [[r[:17] for r in layer] for layer in truth[b]]
    moved = cache.compact()
    used = {p for s in truth for p in cache.pages(s)}
    assert moved > 0 and used == set(range(len(used))) and cache.free_pages == 24 - len(used)
    _holds(cache, truth)
    _fill(cache, cache.extend([b, c, d], [9, 1, 20]), rng, truth)
    _holds(cache, truth)
    for s in list(truth):
        cache.free(s)
    assert cache.free_pages == 24


def test_a_batch_of_another_stream_may_be_dropped_behind_its_calls(torch_gpu, native):
    """Calls on a side stream with batches made on the first one: memory that takes a dropped batch's place is not theirs."""

    from kudacuda_amd.paged_cache import PagedKvCache
    from kudacuda_amd.rotary import rope_frequencies

    cache = PagedKvCache(native, torch, layers=1, kv_heads=2, head_dim=64, num_pages=300)
    freq = torch.from_numpy(rope_frequencies(64, 1e4)[0]).cuda()
    first, second = cache.create(), cache.create()
    q, k, v = (torch.randn((2000, h, 64), device="cuda:0").bfloat16() for h in (4, 2, 2))
    busy = torch.randn((4096, 4096), device="cuda:0")
    batch = cache.extend([first], [2000])
    want = cache.attend(0, batch, cache.append(0, batch, q, k, v, freq))
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(20):
            busy = (busy @ busy).clamp(-1, 1)  # the calls behind it start late
    batch = cache.extend([second], [2000])
    with torch.cuda.stream(side):
        got = cache.attend(0, batch, cache.append(0, batch, q, k, v, freq))
    sizes = [x.numel() * x.element_size() for x in (batch.slots, batch.positions, batch.kv_lens, batch.page_table)]
    del batch
    filled = [torch.full((n,), 0x7f, dtype=torch.uint8, device="cuda:0") for n in sizes for _ in range(8)]
    side.synchronize()
    assert torch.equal(got, want)
    del filled


def test_a_cache_keeps_the_number_of_its_device(torch_gpu, native):
    """"cuda" is the device that is current when the cache is made, not when it is used."""

    from kudacuda_amd.paged_cache import PagedKvCache

    cache = PagedKvCache(native, torch, layers=1, kv_heads=1, head_dim=64, num_pages=2, device="cuda")
    assert cache.device == torch.device("cuda:0") == cache.pool.device
