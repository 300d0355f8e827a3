"""The books of a paged cache and the rotary tables, on the CPU: page copies are made by a stand-in for the library."""

from __future__ import annotations

import contextlib
import ctypes
import math
from types import SimpleNamespace

import numpy as np
import pytest
import torch

from kudacuda_amd._native import Native
from kudacuda_amd.paged_cache import OutOfPages, PagedKvCache
from kudacuda_amd.rotary import rope_frequencies


class StandIn:
    """Copies pages as kudacuda_copy_pages does; keeps the pairs of every call."""

    def __init__(self):
        self.copies = []
        self.cache = None

    def call(self, name, pool, pairs, count, pools, pages, size, page_stride, pool_stride, stream):
        assert name == "kudacuda_copy_pages" and pool == self.cache.pool.data_ptr()
        table = np.ctypeslib.as_array(ctypes.cast(pairs, ctypes.POINTER(ctypes.c_int32)), (count, 2)).copy()
        assert (pools, pages) == self.cache.pool.shape[:2] and page_stride == size and pool_stride == size * pages
        moving = table[table[:, 0] != table[:, 1]]
        assert len(set(table[:, 1])) == count and not set(moving[:, 1]) & set(moving[:, 0])
        self.copies.append([tuple(int(x) for x in p) for p in table])
        self.cache.pool[:, table[:, 1].tolist()] = self.cache.pool[:, table[:, 0].tolist()]


@pytest.fixture
def cache(monkeypatch):
    native = StandIn()
    c = PagedKvCache(native, torch, layers=1, kv_heads=1, head_dim=8, num_pages=10, page_size=4, device="cpu")
    native.cache = c
    monkeypatch.setattr(c, "_stream", lambda: 0)
    return c


def _write(cache, batch, values):
    """Each token's value into its slot's first element."""

    rows = cache.pool[0, :, 0].reshape(-1, cache.head_dim)
    rows[batch.slots, 0] = torch.tensor(values, dtype=rows.dtype)
    cache.pool[0, :, 0] = rows.view(cache.num_pages, cache.page_size, cache.head_dim)


def _read(cache, s):
    rows = cache.pool[0, cache.pages(s), 0, :, 0].flatten()[:cache.length(s)]
    return [int(x) for x in rows]


def test_batches_name_slots_positions_and_tables(cache):
    a, b = cache.create(), cache.create()
    batch = cache.extend([a, b], [5, 3])
    assert cache.pages(a) == [0, 1] and cache.pages(b) == [2] and cache.free_pages == 7
    assert batch.slots.tolist() == [0, 1, 2, 3, 4, 8, 9, 10] and batch.slots.dtype == torch.int64
    assert batch.positions.tolist() == [0, 1, 2, 3, 4, 0, 1, 2]
    assert batch.query_starts.tolist() == [0, 5, 8] and batch.kv_lens.tolist() == [5, 3]
    assert batch.page_table.tolist() == [[0, 1], [2, 0]] and batch.tokens == 8
    assert (batch.max_query_len, batch.max_kv_len) == (5, 5)
    batch = cache.extend([b, a], [2, 0])
    assert batch.slots.tolist() == [11, 12] and batch.positions.tolist() == [3, 4] and cache.pages(b) == [2, 3]
    assert batch.kv_lens.tolist() == [5, 5] and batch.query_starts.tolist() == [0, 2, 2]


def test_a_shared_page_is_copied_by_all_writers_but_its_last(cache):
    a = cache.create()
    _write(cache, cache.extend([a], [6]), range(6))
    b, c = cache.fork(a), cache.fork(a)
    assert cache.free_pages == 8
    _write(cache, cache.extend([a, b, c], [1, 1, 1]), [10, 20, 30])
    assert len(cache.native.copies[0]) == 2 and cache.free_pages == 6
    assert [_read(cache, s) for s in (a, b, c)] == [[0, 1, 2, 3, 4, 5, x] for x in (10, 20, 30)]
    # a full last page is shared on: nothing to copy
    _write(cache, cache.extend([a], [1]), [11])
    d = cache.fork(a)
    _write(cache, cache.extend([d, a], [1, 1]), [40, 12])
    assert len(cache.native.copies) == 1
    assert _read(cache, d)[-3:] == [10, 11, 40] and _read(cache, a)[-3:] == [10, 11, 12]
    # a reader keeps a shared page while the writer copies it
    e = cache.fork(d)
    _write(cache, cache.extend([d], [1]), [41])
    assert _read(cache, e)[-1] == 40 and _read(cache, d)[-2:] == [40, 41]


def test_too_few_pages_change_nothing(cache):
    a = cache.create()
    cache.extend([a], [30])
    b = cache.fork(a)
    state = (cache.free_pages, cache.pages(a), cache.length(a), cache.pages(b))
    for sequences, counts in (([a], [11]), ([a, b], [1, 10]), ([b], [14])):
        with pytest.raises(OutOfPages):
            cache.extend(sequences, counts)
        assert (cache.free_pages, cache.pages(a), cache.length(a), cache.pages(b)) == state
    assert cache.native.copies == []
    cache.extend([a, b], [2, 2])  # a's copy of the shared page, b keeps it
    assert cache.free_pages == 1


def test_free_truncate_and_compact(cache):
    a, b, c = (cache.create() for _ in range(3))
    _write(cache, cache.extend([a, b, c], [7, 9, 5]), list(range(7)) + list(range(50, 59)) + list(range(90, 95)))
    d = cache.fork(c)
    cache.free(a)
    cache.truncate(b, 4)
    assert cache.free_pages == 10 - 1 - 2
    assert cache.compact() == 2 and cache.native.copies[-1] == [(5, 0), (6, 1)]
    assert cache.pages(b) == [2] and cache.pages(c) == cache.pages(d) == [0, 1]
    assert _read(cache, b) == [50, 51, 52, 53] and _read(cache, c) == _read(cache, d) == [90, 91, 92, 93, 94]
    assert cache.compact() == 0 and len(cache.native.copies) == 1
    assert cache.extend([b], [1]).slots.tolist() == [12]
    for s in (b, c, d):
        cache.free(s)
    assert cache.free_pages == 10 and sorted(cache._free) == list(range(10))
    with pytest.raises(KeyError):
        cache.length(b)


def test_requests_that_make_no_sense_are_refused(cache):
    a = cache.create()
    for sequences, counts in (([a, a], [1, 1]), ([], []), ([a], [0]), ([a], [-1]), ([a], [1, 2])):
        with pytest.raises(ValueError):
            cache.extend(sequences, counts)
    with pytest.raises(KeyError):
        cache.extend([a, 77], [1, 1])
    with pytest.raises(ValueError):
        cache.truncate(a, 1)
    for bad in (dict(page_size=12), dict(page_size=8192), dict(num_pages=0), dict(head_dim=12), dict(dtype=torch.float32)):
        with pytest.raises(ValueError):
            PagedKvCache(StandIn(), torch, **(dict(layers=1, kv_heads=1, head_dim=8, num_pages=4, device="cpu") | bad))
    batch = cache.extend([a], [2])
    rows = torch.zeros((2, 1, 8), dtype=torch.bfloat16)
    freq = torch.zeros(4, dtype=torch.float64)
    for q, k, f in ((rows[:1], rows, freq), (rows, rows.float(), freq), (rows, rows.expand(2, 3, 8), freq),
                    (rows, rows, freq.float()), (torch.zeros((2, 8, 2), dtype=torch.bfloat16).transpose(1, 2), rows, freq)):
        with pytest.raises(ValueError):
            cache.append(0, batch, q, k, rows, f)


def test_random_use_keeps_every_sequence(cache):
    """Forks, frees, truncations and compactions at random, against plain lists."""

    rng = np.random.default_rng(5)
    truth, value = {}, 0
    for _ in range(600):
        what = rng.integers(0, 8)
        live = list(truth)
        if what == 0 or not live:
            truth[cache.create()] = []
        elif what == 1 and len(live) < 6:
            s = live[rng.integers(len(live))]
            truth[cache.fork(s)] = list(truth[s])
        elif what == 2:
            s = live[rng.integers(len(live))]
            cache.free(s)
            del truth[s]
        elif what == 3:
            s = live[rng.integers(len(live))]
            n = int(rng.integers(0, len(truth[s]) + 1))
            cache.truncate(s, n)
            truth[s] = truth[s][:n]
        elif what == 4:
            cache.compact()
        else:
            some = [s for s in live if rng.random() < 0.7] or live[:1]
            counts = [int(rng.integers(0, 5)) for _ in some]
            if sum(counts) == 0:
                continue
            try:
                batch = cache.extend(some, counts)
            except OutOfPages:
                continue
            new = [(value + i) % 251 for i in range(sum(counts))]
            value += len(new)
            _write(cache, batch, new)
            for s, c in zip(some, counts):
                truth[s] += new[:c]
                new = new[c:]
        assert {s: _read(cache, s) for s in truth} == truth
        assert cache.free_pages == 10 - len({p for s in truth for p in cache.pages(s)})


# ------------------------------------------------------------- rotary tables
def test_rotary_frequencies():
    plain, one = rope_frequencies(128, 1.0e6)
    assert one == 1.0 and plain[0] == 1.0 and len(plain) == 64
    assert plain[-1] == pytest.approx(1.0e6 ** (-126 / 128), rel=1e-15)
    assert np.allclose(rope_frequencies(128, scaling="linear", factor=4.0)[0], plain / 4.0, rtol=1e-15)
    ntk = rope_frequencies(128, scaling="ntk", factor=8.0)[0]
    assert ntk[0] == 1.0 and ntk[-1] == pytest.approx(plain[-1] / 8.0, rel=1e-12)
    yarn, amplitude = rope_frequencies(128, scaling="yarn", factor=16.0, original_positions=4096)
    turns = 4096 * plain / (2 * math.pi)
    assert amplitude == pytest.approx(0.1 * math.log(16.0) + 1.0)
    assert np.array_equal(yarn[turns > 32], plain[turns > 32]) and np.allclose(yarn[turns < 1], plain[turns < 1] / 16.0)
    between = (turns > 1) & (turns < 32)
    assert between.any() and (yarn[between] < plain[between]).all() and (yarn[between] > plain[between] / 16.0).all()
    for scaling in ("none", "linear", "ntk", "yarn"):
        assert np.allclose(rope_frequencies(64, scaling=scaling)[0], rope_frequencies(64)[0], rtol=1e-12)


@pytest.mark.parametrize("bad", [dict(rotary_dim=3), dict(rotary_dim=0), dict(scaling="other"), dict(factor=0.5),
                                 dict(theta=-1.0), dict(factor=float("nan"))])
def test_rotary_refusals(bad):
    with pytest.raises(ValueError):
        rope_frequencies(**(dict(rotary_dim=64) | bad))


@pytest.mark.parametrize("device", ["cpu", "cuda:1"])
def test_a_cache_lies_on_its_handles_device(device):
    native = Native.__new__(Native)
    native.handle, native.device_id = None, 0
    with pytest.raises(ValueError, match="cuda:0"):
        PagedKvCache(native, torch, layers=1, kv_heads=1, head_dim=8, num_pages=1, device=device)


@pytest.mark.parametrize("fault", ["copy", "upload"])
def test_an_extension_that_fails_changes_nothing(cache, monkeypatch, fault):
    """A refused page copy, or a batch that finds no device memory: the books are as before, and a retry is right."""

    a, b = cache.create(), cache.create()
    _write(cache, cache.extend([a, b], [6, 3]), list(range(9)))
    c = cache.fork(a)

    def state():
        return [(cache.pages(s), cache.length(s)) for s in (a, b, c)], list(cache._free), list(cache._users)

    before = state()
    with monkeypatch.context() as m:
        def fail(*_args):
            raise RuntimeError("out of device memory")

        if fault == "copy":
            m.setattr(cache.native, "call", fail)
        else:
            m.setattr(cache.torch, "from_numpy", fail)
        with pytest.raises(RuntimeError, match="memory"):
            cache.extend([b, a], [2, 3])
    assert state() == before
    _write(cache, cache.extend([b, a], [2, 3]), [20, 21, 10, 11, 12])
    assert [_read(cache, s) for s in (a, b, c)] == [[*range(6), 10, 11, 12], [6, 7, 8, 20, 21], list(range(6))]


@pytest.mark.parametrize("dim,theta,factor,positions,slow,fast", [
    (128, 1.0e6, 4.0, 32768, 1.0, 32.0), (64, 1.0e4, 16.0, 4096, 1.0, 32.0), (96, 5.0e5, 8.0, 8192, 1.0, 32.0),
    (32, 1.0e4, 40.0, 4096, 1.0, 32.0), (128, 1.0e6, 2.0, 32768, 2.0, 8.0), (64, 1.0e4, 4.0, 100, 1.0, 32.0),
    (8, 1.0e4, 4.0, 1 << 20, 1.0, 1.5), (128, 1.0e4, 1.0, 4096, 1.0, 32.0)])
def test_yarn_frequencies_are_those_that_models_run(dim, theta, factor, positions, slow, fast):
    """Transformers' table, which is made in fp32: powers and exponents off by 2^-21 (14 of them at 2^-25), sums by a
    few roundings, and 1 - ramp by 2^-24 of the plain frequency, up to `factor` times the sum."""

    transformers = pytest.importorskip("transformers")
    from transformers.modeling_rope_utils import ROPE_INIT_FUNCTIONS

    scaling = dict(rope_type="yarn", rope_theta=theta, factor=factor, original_max_position_embeddings=positions,
                   beta_slow=slow, beta_fast=fast)
    config = transformers.Qwen2Config(hidden_size=4 * dim, num_attention_heads=4, num_key_value_heads=4,
                                      max_position_embeddings=int(positions * factor), rope_parameters=scaling)
    want, scale = ROPE_INIT_FUNCTIONS["yarn"](config, "cpu")
    got, amplitude = rope_frequencies(dim, theta, scaling="yarn", factor=factor, original_positions=positions, slow=slow,
                                      fast=fast)
    assert amplitude == pytest.approx(scale, rel=1e-6)
    want = want.double().numpy()
    assert (np.abs(got - want) <= (2.0**-20 + factor * 2.0**-23) * want).all(), (got / want).tolist()


def test_yarn_keeps_pairs_that_all_turn_often():
    plain = rope_frequencies(8, 1.0e4)[0]
    assert np.array_equal(rope_frequencies(8, 1.0e4, scaling="yarn", factor=4.0, original_positions=1 << 40)[0], plain)


@pytest.mark.parametrize("bad", [dict(slow=32.0, fast=1.0), dict(slow=0.0), dict(original_positions=0), dict(theta=1.0)])
def test_yarn_refusals(bad):
    with pytest.raises(ValueError):
        rope_frequencies(**(dict(rotary_dim=64, scaling="yarn", factor=4.0) | bad))


# -------------------------------------------------- streams and devices of the calls
class FakeCuda:
    """torch.cuda with two devices of one stream each; `capturing` are those whose stream a graph captures."""

    def __init__(self):
        self.current = 0
        self.capturing = set()

    def current_device(self):
        return self.current

    def current_stream(self, device):
        return SimpleNamespace(cuda_stream=100 + torch.device(device).index)

    def is_current_stream_capturing(self):
        return self.current in self.capturing

    @contextlib.contextmanager
    def device(self, device):
        before, self.current = self.current, torch.device(device).index
        yield
        self.current = before


@pytest.fixture
def second(monkeypatch):
    """A cache on cuda:1 (its tensors stay on the CPU) and its torch; calls are kept."""

    calls = []
    native = SimpleNamespace(call=lambda name, *args: calls.append((name, args)),
                             lib=SimpleNamespace(kudacuda_paged_attention_workspace_bytes=lambda *_: 64))
    c = PagedKvCache(native, torch, layers=1, kv_heads=1, head_dim=8, num_pages=4, page_size=4, device="cpu")
    cuda = FakeCuda()
    c.torch = SimpleNamespace(cuda=cuda, empty=lambda n, dtype, device: torch.empty(n, dtype=dtype), uint8=torch.uint8,
                              empty_like=torch.empty_like, contiguous_format=torch.contiguous_format,
                              from_numpy=torch.from_numpy, float64=torch.float64, bfloat16=torch.bfloat16)
    monkeypatch.setattr(c, "_stream", lambda: 101)
    batch = c.extend([c.create()], [1])
    c.device = torch.device("cuda:1")
    return c, cuda, batch, calls


def test_a_captured_call_has_its_own_workspace_whichever_device_is_current(second):
    cache, cuda, batch, calls = second
    q = torch.zeros((1, 1, 8), dtype=torch.bfloat16)
    cuda.capturing = {1}
    for current in (0, 1):
        cuda.current = current
        cache.attend(0, batch, q)
        assert cache._workspaces == {} and cuda.current == current
    cuda.capturing = {0}  # another device's graph: an ordinary call here
    for current in (0, 1):
        cuda.current = current
        cache.attend(0, batch, q)
    assert list(cache._workspaces) == [101]
    kept = cache._workspaces[101].data_ptr()
    assert [args[7] == kept for _, args in calls][-2:] == [True, True]


def test_one_token_has_no_stride(second):
    """The row of a single token may lie anywhere on its boundary: its distance to a next one is never used."""

    cache, _, batch, calls = second
    rows = torch.zeros(3 * 17, dtype=torch.bfloat16)
    q = torch.as_strided(rows, (1, 2, 8), (17, 8, 1))
    k = torch.as_strided(rows, (1, 1, 8), (3, 8, 1))
    cache.append(0, batch, q, k, k, torch.zeros(4, dtype=torch.float64), out=q)
    cache.attend(0, batch, q)
    append, attend = (args for _, args in calls)
    assert append[16:20] == (16, 8, 8, 16) and attend[17:19] == (16, 16)
