"""GPU: adapters of many requests beside a projection (kudacuda_lora_add) against products in 64 bits."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from kudacuda_amd.lora import LoraAdapters, lora_batch
from tests._paged_ref import CODE, HALF, f64

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16


class Round:
    """Requests with adapters of these ranks (None: none) and their rows."""

    def __init__(self, native, seed, chunks, ranks, inner, outer, *, dtype=BF16, max_rank=None, gap=0, spare=2):
        rng = np.random.default_rng([91, seed])
        self.native, self.dtype, self.chunks, self.ranks = native, dtype, chunks, ranks
        self.inner, self.outer, self.gap = inner, outer, gap
        used = sorted({r for r in ranks if r is not None})
        self.pool = LoraAdapters(native, torch, in_features=inner, out_features=outer, adapters=len(ranks) + spare,
                                 max_rank=max_rank or max([1] + [r for _, r in used]), dtype=dtype)
        for x in (self.pool.a, self.pool.b):
            x.fill_(float("nan"))  # what no adapter owns must not be met
        normal = lambda *s: torch.from_numpy(rng.standard_normal(s).astype(np.float32))  # noqa: E731
        self.factors = {}
        for name, rank in used:
            a, b = (normal(rank, inner) / inner**0.5).to(dtype), (normal(outer, rank) * 0.3).to(dtype)
            scale = float(np.float32(rng.uniform(0.5, 2.0)))
            self.pool.load(name, a, b, scale)
            self.factors[name] = f64(a), f64(b), scale
        tokens = sum(chunks)
        self.x, self.base = normal(tokens, inner).to(dtype), normal(tokens, outer).to(dtype)
        self.batch = lora_batch(torch, [None if r is None else r[0] for r in ranks], chunks)

    def rows(self, x):
        """On the device, ``gap`` elements between rows."""

        out = torch.full((x.shape[0], x.shape[1] + self.gap), 7.25, dtype=self.dtype, device="cuda:0")
        out[:, :x.shape[1]] = x.cuda()
        return out[:, :x.shape[1]]

    def want(self, base=True):
        """(out, bound).  u = x A^T: fp32 sums of depth in / 128 + 68 at most (a wave's steps, 32 products of each, four
        waves, 32 shares), each rounding by 2^-24 of sum |x a|; its two parts are off by 2^-17 (bf16), 2^-22 (fp16) of
        its row's largest (or less); the second product sums up to 2 * 128 of them, by 2^-24 each."""

        out, bound = f64(self.base) * base, np.zeros((sum(self.chunks), self.outer))
        parts = 2.0**-17 if self.dtype == BF16 else 2.0**-22
        at = 0
        for n, r in zip(self.chunks, self.ranks):
            if r is not None:
                a, b, scale = self.factors[r[0]]
                x = f64(self.x[at:at + n])
                u = x @ a.T
                out[at:at + n] += scale * u @ b.T
                off = (self.inner / 128 + 68) * 2.0**-24 * (np.abs(x) @ np.abs(a).T)
                off += (parts + 256 * 2.0**-24) * np.abs(u).max(axis=1, keepdims=True)
                bound[at:at + n] = scale * off @ np.abs(b).T
            at += n
        return out, bound + HALF[self.dtype] * np.abs(out) + 2.0**-23 * np.abs(f64(self.base)) + 2.0**-25

    def check(self, got, base=True):
        want, bound = self.want(base)
        off = np.abs(f64(got) - want)
        assert (off <= bound).all(), float(np.nanmax(off / bound))


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("chunks,ranks,inner,outer,max_rank", [
    ([1], [(0, 16)], 2048, 2048, None),
    ([1], [(0, 1)], 8, 8, 8),
    ([1, 1, 1], [(0, 8), (1, 8), (0, 8)], 264, 1000, 8),
    ([1] * 20, [(i % 7, (8, 16, 24, 32, 64, 5, 1)[i % 7]) for i in range(20)], 512, 328, None),
    ([16], [(0, 16)], 2048, 256, None),
    ([17], [(1, 40)], 136, 264, 64),
    ([64, 65, 63], [(0, 32), (1, 16), (2, 33)], 256, 512, 64),
    ([300, 1, 40], [(0, 64), None, (1, 128)], 640, 72, None),
    ([5, 200], [None, (3, 100)], 1000, 4096, 128),
    ([3, 2], [None, None], 64, 64, 16),
    ([700], [(0, 16)], 11008, 2048, None),
    ([2, 3, 2], [(1, 8), (0, 16), (1, 8)], 32, 40, 96),
    ([1] * 300, [(i % 50, 12) for i in range(300)], 128, 64, None),
    ([129] * 9, [(i, 16) for i in range(9)], 2048, 2560, None),
    # few rows a tile: one launch where factors and blocks are few, two otherwise
    ([40, 1, 1, 1, 2], [(0, 24), (1, 8), (2, 3), (3, 16), None], 2048, 520, None),
    ([40, 1, 1, 1, 2], [(0, 24), (1, 8), (2, 3), (3, 16), None], 11008, 520, None),
    ([1, 4, 1], [(0, 64), (1, 50), (2, 33)], 1024, 1000, None),
    ([1, 4, 1], [(0, 64), (1, 50), (2, 33)], 1032, 1000, None),
    ([2, 1, 33], [(0, 128), (1, 100), (2, 65)], 520, 264, None),
])
def test_matches_fp64(torch_gpu, native, dtype, chunks, ranks, inner, outer, max_rank):
    print(f"adapters {ranks[:9]} for {chunks[:9]} rows, {inner} -> {outer}, {dtype}", flush=True)
    r = Round(native, 1, chunks, ranks, inner, outer, dtype=dtype, max_rank=max_rank)
    x, base = r.rows(r.x), r.rows(r.base)
    out = torch.full_like(base, 7.25)
    r.check(r.pool.add(r.batch, x, base, out))
    assert torch.equal(base.cpu(), r.base)
    assert torch.equal(r.pool.add(r.batch, x, base), out) and torch.equal(base, out)  # in place: the same


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_rows_with_gaps_and_no_base(torch_gpu, native, dtype):
    r = Round(native, 2, [3, 70, 1], [(0, 16), (1, 20), None], 200, 104, dtype=dtype, gap=8)
    x, base = r.rows(r.x), r.rows(r.base)
    r.check(r.pool.add(r.batch, x, base))
    whole = torch.as_strided(base, (74, 112), (112, 1))
    assert (whole[:, 104:] == 7.25).all()
    out = torch.full((74, 104), 7.25, dtype=dtype, device="cuda:0")
    _call(native, r, x, 0, out)
    r.check(out, base=False)
    assert (out[73] == 0).all()


def _call(native, r, x, base, out, order=None, tiles=None, tokens=None, workspace=None):
    order, tiles = r.batch.order if order is None else order, r.batch.tiles if tiles is None else tiles
    p, tokens = r.pool, r.batch.tokens if tokens is None else tokens
    nbytes = native.lib.kudacuda_lora_workspace_bytes(tokens, tiles.shape[0], p.max_rank, p.in_features)
    workspace = torch.empty(nbytes, dtype=torch.uint8, device="cuda:0") if workspace is None else workspace
    native.call("kudacuda_lora_add", x.data_ptr(), p.a.data_ptr(), p.b.data_ptr(), p.ranks.data_ptr(), p.scales.data_ptr(),
                order.data_ptr(), tiles.data_ptr(), base if isinstance(base, int) else base.data_ptr(), out.data_ptr(),
                workspace.data_ptr(), nbytes, CODE[r.dtype], tokens, tiles.shape[0], p.count, p.max_rank, p.in_features,
                p.out_features, x.stride(0), 0 if isinstance(base, int) else base.stride(0), out.stride(0),
                torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    return workspace


def test_plans_that_name_too_much_stay_inside(torch_gpu, native):
    """Tiles and rows outside the round are left out, adapters outside the pool add nothing, the workspace's end holds."""

    r = Round(native, 3, [20, 40], [(0, 16), (1, 8)], 256, 128)
    x, base = r.rows(r.x), r.rows(r.base)
    want, bound = r.want()
    up = lambda rows: torch.tensor(rows, dtype=torch.int32, device="cuda:0")  # noqa: E731
    order = r.batch.order.clone()
    order[[2, 30]] = up([-1, 60])  # rows 2 and 30 are named by nobody
    tiles = up([[0, 0, 20], [99, 20, 5], [-3, 25, 3], [1, 28, 2**31 - 1], [0, -5, 64], [1, 60, 3], [0, 2**31 - 1, 9], [0, 3, -2]])
    out = torch.full_like(base, 7.25)
    nbytes = native.lib.kudacuda_lora_workspace_bytes(60, 8, r.pool.max_rank, 256)
    workspace = torch.full((nbytes + 4096,), 0x7f, dtype=torch.uint8, device="cuda:0")
    _call(native, r, x, base, out, order, tiles, workspace=workspace)
    got = f64(out)
    assert (workspace[nbytes:] == 0x7f).all() and (got[[2, 30]] == 7.25).all()
    rows = [i for i in range(60) if i not in (2, 30) and not 20 <= i < 28]
    assert (np.abs(got - want) <= bound)[rows].all()
    assert np.array_equal(got[20:28], f64(r.base[20:28]))


def test_ranks_outside_the_pool_are_cut(torch_gpu, native):
    r = Round(native, 4, [3, 2, 4], [(0, 16), (1, 16), (2, 16)], 64, 64)
    x, base = r.rows(r.x), r.rows(r.base)
    r.pool.ranks[0], r.pool.ranks[1] = 1 << 30, -7
    want, bound = r.want()
    out = r.pool.add(r.batch, x, base, torch.empty_like(base))
    keep = [0, 1, 2, 5, 6, 7, 8]
    assert (np.abs(f64(out) - want) <= bound)[keep].all() and np.array_equal(f64(out[3:5]), f64(r.base[3:5]))


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_inner_rows_of_any_size(torch_gpu, native, dtype):
    """Rows whose x A^T lies far below and above fp16's range keep their bits."""

    r = Round(native, 5, [6], [(0, 8)], 64, 32, dtype=dtype)
    size = torch.tensor([2.0**-14, 2.0**-6, 1.0, 2.0**5, 2.0**9, 2.0**12]).to(dtype)[:, None]
    r.x = (r.x * size).to(dtype)
    a, b, _ = r.factors[0]
    big = 16.0
    r.pool.load(0, torch.from_numpy(a * big), torch.from_numpy(b / 64), 2.0**-6)
    r.factors[0] = f64(r.pool.a[0, :8]), f64(r.pool.b[0, :32 * 8].view(32, 8)), 2.0**-6
    r.base.zero_()
    r.check(r.pool.add(r.batch, r.rows(r.x), r.rows(r.base)))


def test_infinite_inputs_reach_their_own_row_only(torch_gpu, native):
    r = Round(native, 6, [5, 5], [(0, 16), (0, 16)], 64, 64)
    r.x[3, 7] = float("inf")
    r.x[4, 9] = float("nan")
    out = f64(r.pool.add(r.batch, r.rows(r.x), r.rows(r.base)))
    assert not np.isfinite(out[[3, 4]]).any()
    r.x[3, 7] = r.x[4, 9] = 0
    want, bound = r.want()
    rows = [0, 1, 2, 5, 6, 7, 8, 9]
    assert (np.abs(out - want) <= bound)[rows].all()


def test_captured_calls_follow_their_plan(torch_gpu, native):
    """Two graphs on two streams, each with a workspace of its own; a plan that changes in place is read at replay."""

    rounds = [Round(native, 7 + i, [1] * 40, [(j % 5, 16) for j in range(40)], 1024, 512) for i in range(2)]
    rows = [(r.rows(r.x), r.rows(r.base)) for r in rounds]
    outs = [torch.zeros_like(b) for _, b in rows]
    torch.cuda.synchronize()
    graphs, streams = [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for r, (x, base), out, s in zip(rounds, rows, outs, streams):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=s):
            r.pool.add(r.batch, x, base, out)
    for turn in range(6):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        for s in streams:
            s.synchronize()
        for r, out, (x, base) in zip(rounds, outs, rows):
            r.check(out)
            assert torch.equal(r.pool.add(r.batch, x, base, torch.empty_like(base)), out)
        torch.cuda.synchronize()
        r = rounds[0]
        ranks = [(int(j), 16) for j in np.random.default_rng(turn).integers(0, 5, 40)]
        plan = lora_batch(torch, [j for j, _ in ranks], [1] * 40)
        if plan.tile_count == r.batch.tile_count:
            r.ranks = ranks
            r.batch.order.copy_(plan.order)
            r.batch.tiles.copy_(plan.tiles)
            torch.cuda.synchronize()


def test_calls_on_another_stream_and_again(torch_gpu, native):
    r = Round(native, 9, [100, 30], [(0, 64), (1, 8)], 2048, 1024)
    x, base = r.rows(r.x), r.rows(r.base)
    want = r.pool.add(r.batch, x, base, torch.empty_like(base))
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        got = [r.pool.add(r.batch, x, base, torch.empty_like(base)) for _ in range(3)]
    side.synchronize()
    assert all(torch.equal(g, want) for g in got)
    r.check(want)


def test_the_class_refuses_rows_that_do_not_fit(torch_gpu, native):
    r = Round(native, 10, [3], [(0, 8)], 64, 32)
    x, base = r.rows(r.x), r.rows(r.base)
    for bad in ((x[:2], base), (x, base[:, :24]), (x.half(), base), (x.cpu(), base), (x, base, base.t().contiguous().t())):
        with pytest.raises(ValueError):
            r.pool.add(r.batch, *bad)


def test_trained_factors_and_adapters_that_are_not_there(torch_gpu, native):
    """Parameters are loaded as they are, without a graph behind them; a plan may not name more than there are."""

    pool = LoraAdapters(native, torch, in_features=64, out_features=32, adapters=2, max_rank=8)
    a, b = (torch.randn(s, device="cuda:0").bfloat16().requires_grad_() for s in ((4, 64), (32, 4)))
    pool.load(1, a, b, scale=2.0)
    x, y = torch.randn((3, 64), device="cuda:0").bfloat16(), torch.zeros((3, 32), dtype=BF16, device="cuda:0")
    pool.add(lora_batch(torch, [1], [3]), x, y)
    assert not (pool.a.requires_grad or pool.b.requires_grad) and int(y.count_nonzero()) > 0
    before = y.clone()
    with pytest.raises(IndexError):
        pool.add(lora_batch(torch, [0, 2], [1, 2]), x, y)
    assert torch.equal(y, before)
