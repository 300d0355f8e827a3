"""CPU: the host form of the microscaled numbers that the GPU tests compare with, and the cache's own refusals."""

from __future__ import annotations

from types import SimpleNamespace

import numpy as np
import pytest
import torch

from kudacuda_amd._native import Native
from kudacuda_amd.lora import LoraAdapters, lora_batch
from kudacuda_amd.paged_cache import PagedKvCache
from tests import _mx_ref as mx

NATIVE = SimpleNamespace()


def test_levels():
    assert list(mx.levels(4)[:8]) == [0, 0.5, 1, 1.5, 2, 3, 4, 6] and (mx.levels(4)[8:] == -mx.levels(4)[:8]).all()
    ours, theirs = mx.levels(8), torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(ours, theirs, equal_nan=True)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_nothing_is_off_by_more_than_half_a_step(bits, dtype):
    """Up to where the type ends, and every held number is one of the type."""

    rng = np.random.default_rng(bits)
    low, high = mx.exponents(bits, dtype)
    x = torch.from_numpy(rng.standard_normal((400, 64)) * 2.0 ** rng.integers(low, high + 2, (400, 1))).to(dtype).double().numpy()
    codes, blocks = mx.pack(x, bits, dtype)
    held = mx.unpack(codes, blocks, bits)
    mx.numbers(held, dtype)
    power = np.repeat(2.0 ** (blocks.astype(np.float64) - 127), 32, axis=-1)
    m = np.abs(x) / power
    lowest = 0 if bits == 4 else -6
    step = 2.0 ** (np.floor(np.log2(np.maximum(m, 2.0**lowest))) - (1 if bits == 4 else 3))
    assert (np.abs(held - x) / power <= step / 2).all()
    # the next lower exponent would not do
    top = np.abs(x).reshape(400, 2, 32).max(axis=-1)
    spare = blocks.astype(int) - 127 > low
    assert (top[spare] >= (7.0 if bits == 4 else 464.0) * 2.0 ** (blocks[spare].astype(np.float64) - 128)).all()


def test_blocks_without_a_number_and_without_a_size():
    x = np.zeros((3, 64))
    x[0, 5], x[1, 40], x[2, 0] = np.nan, np.inf, 2.0**-130
    for bits in (4, 8):
        codes, blocks = mx.pack(x, bits, torch.bfloat16)
        assert blocks.tolist() == [[255, 17], [17, 255], [17, 17]]
        held = mx.unpack(codes, blocks, bits)
        assert np.isnan(held[0, :32]).all() and np.isnan(held[1, 32:]).all() and (held[2] == 0).all()


@pytest.mark.parametrize("bits", [4, 8])
def test_pages_there_and_back(bits):
    rng = np.random.default_rng(3)
    codes, blocks = rng.integers(0, 1 << bits, (5, 3, 16, 64), dtype=np.uint8), rng.integers(0, 256, (5, 3, 16, 2), dtype=np.uint8)
    data = mx.to_pages(codes, blocks, bits, extra=32)
    assert data.shape[1] == mx.page_bytes(3, 16, 64, bits) + 32
    a, b = mx.from_pages(data, 3, 16, 64, bits)
    assert np.array_equal(a, codes) and np.array_equal(b, blocks)


@pytest.mark.parametrize("bad", [dict(bits=5), dict(bits=4, head_dim=96), dict(bits=8, head_dim=256), dict(bits=4, page_size=8),
                                 dict(bits=4, kv_heads=2048)])
def test_cache_refusals(bad):
    with pytest.raises(ValueError):
        PagedKvCache(NATIVE, torch, **(dict(layers=1, kv_heads=2, head_dim=64, num_pages=4, device="cpu") | bad))


def test_a_cache_of_fewer_bits_takes_less():
    sizes = {b: PagedKvCache(NATIVE, torch, layers=2, kv_heads=2, head_dim=128, num_pages=8, bits=b, device="cpu").pool.nbytes
             for b in (16, 8, 4)}
    assert sizes[16] == 2 * 2 * 8 * 16 * 2 * 256 and sizes[8] * 2 * 128 == sizes[16] * 132 and sizes[4] * 4 * 64 == sizes[16] * 68


def test_reading_past_a_sequence_is_refused():
    cache = PagedKvCache(NATIVE, torch, layers=1, kv_heads=2, head_dim=64, num_pages=4, bits=4, device="cpu")
    s = cache.create()
    for start, stop in ((0, 1), (-1, 0), (1, 0)):
        with pytest.raises(ValueError):
            cache.read(0, s, start, stop)
    with pytest.raises(KeyError):
        cache.read(0, s + 1)


# ------------------------------------------------------------------ adapters
def test_a_plan_lists_every_row_once_in_tiles_of_one_adapter():
    batch = lora_batch(torch, [2, None, 0, 2, 5, 7], [3, 70, 64, 100, 0, 1], device="cpu")
    rows = np.repeat([2, -1, 0, 2, 5, 7], [3, 70, 64, 100, 0, 1])
    order, tiles = batch.order.numpy(), batch.tiles.numpy()
    assert sorted(order) == list(range(238)) and batch.tokens == 238 and batch.tile_count == len(tiles)
    at = 0
    for adapter, first, count in tiles:
        assert first == at and 1 <= count <= 64 and (rows[order[first:first + count]] == adapter).all()
        at += count
    assert at == 238 and len(tiles) == 2 + 1 + 2 + 1


@pytest.mark.parametrize("adapters,counts", [([], []), ([0], [0]), ([0, 1], [1]), ([-2], [1]), ([0], [-1])])
def test_plan_refusals(adapters, counts):
    with pytest.raises(ValueError):
        lora_batch(torch, adapters, counts, device="cpu")


@pytest.mark.parametrize("bad", [dict(max_rank=0), dict(max_rank=129), dict(adapters=0), dict(in_features=36), dict(out_features=4),
                                 dict(dtype=torch.float32)])
def test_adapter_refusals(bad):
    with pytest.raises(ValueError):
        LoraAdapters(NATIVE, torch, **(dict(in_features=32, out_features=64, adapters=2, max_rank=8, device="cpu") | bad))


def test_factors_lie_in_rows_of_their_rank():
    pool = LoraAdapters(NATIVE, torch, in_features=16, out_features=24, adapters=3, max_rank=20, device="cpu")
    assert pool.max_rank == 24
    a, b = torch.randn(5, 16), torch.randn(24, 5)
    pool.b.fill_(7)
    pool.load(1, a, b, 0.25)
    assert torch.equal(pool.a[1, :5], a.bfloat16()) and pool.ranks.tolist() == [0, 5, 0] and float(pool.scales[1]) == 0.25
    rows = pool.b[1, :24 * 8].view(24, 8)
    assert torch.equal(rows[:, :5], b.bfloat16()) and (rows[:, 5:] == 0).all() and (pool.b[0] == 7).all()
    pool.clear(1)
    assert pool.ranks.tolist() == [0, 0, 0]
    for index, x, y in ((1, torch.randn(25, 16), torch.randn(24, 25)), (1, torch.randn(5, 15), b), (1, a, b.T), (1, a[0], b)):
        with pytest.raises(ValueError):
            pool.load(index, x, y)
    with pytest.raises(IndexError):
        pool.load(3, a, b)


@pytest.mark.parametrize("device", ["cpu", "cuda:1"])
def test_adapters_lie_on_their_handles_device(device):
    native = Native.__new__(Native)
    native.handle, native.device_id = None, 0
    with pytest.raises(ValueError, match="cuda:0"):
        LoraAdapters(native, torch, in_features=8, out_features=8, adapters=1, max_rank=8, device=device)


def test_a_plan_of_another_device_or_of_more_adapters_is_refused():
    pool = LoraAdapters(None, torch, in_features=8, out_features=8, adapters=2, max_rank=8, device="cpu")
    x, y = torch.zeros((3, 8), dtype=torch.bfloat16), torch.zeros((3, 8), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="plan on meta"):
        pool.add(lora_batch(torch, [1], [3], device="meta"), x, y)
    with pytest.raises(IndexError):
        pool.add(lora_batch(torch, [2], [3], device="cpu"), x, y)
