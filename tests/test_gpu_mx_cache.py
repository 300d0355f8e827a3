"""GPU: rows into and out of a cache of 8 or 4 bits, byte for byte against the host form."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from kudacuda_amd.paged_cache import PagedKvCache
from kudacuda_amd.rotary import rope_frequencies
from tests import _mx_ref as mx
from tests._paged_ref import CODE, HALF, f64, rope, rope_bound

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16


class Append:
    """Tokens on their way into pages of which only some are theirs."""

    def __init__(self, seed, tokens, *, heads=4, kv_heads=2, dim=64, rotary=None, pairs=False, page=16, bits=4, dtype=BF16,
                 amplitude=1.0, gap=0, extra=0, padding=(), offset=0):
        rng = np.random.default_rng([seed, tokens])
        self.tokens, self.heads, self.kv_heads, self.dim, self.page = tokens, heads, kv_heads, dim, page
        self.rotary, self.pairs, self.bits, self.dtype = rotary or dim, pairs, bits, dtype
        self.amplitude = float(np.float32(amplitude))
        self.num_pages = -(-tokens // page) + 3
        places = rng.permutation(self.num_pages * page)[:tokens].astype(np.int64)
        for i, slot in padding:
            places[i] = slot
        self.slots = places
        self.positions = rng.integers(0, 130000, tokens).astype(np.int32)
        self.freq = rope_frequencies(self.rotary, 1e6)[0]
        width = (heads + 2 * kv_heads) * dim
        spread = np.exp(rng.standard_normal(width) * 0.7) * 2.0 ** rng.integers(-3, 4, (tokens, 1))
        data = torch.from_numpy((rng.standard_normal((tokens, width)) * spread).astype(np.float32)).to(dtype)
        self.row = width + gap
        self.data = torch.zeros(tokens * self.row + offset, dtype=dtype)[offset:].view(tokens, self.row)
        self.data[:, :width] = data
        self.qkv = data
        self.extra, self.offset = extra, offset
        self.page_bytes = mx.page_bytes(kv_heads, page, dim, bits) + extra

    def parts(self):
        h, g = self.heads, self.kv_heads
        return f64(self.qkv).reshape(self.tokens, h + 2 * g, self.dim)[:, :h], f64(self.qkv).reshape(
            self.tokens, h + 2 * g, self.dim)[:, h:h + g], f64(self.qkv).reshape(self.tokens, h + 2 * g, self.dim)[:, h + g:]

    def call(self, native, in_place=False):
        qkv = torch.zeros(self.tokens * self.row + self.offset, dtype=self.dtype, device="cuda:0")[self.offset:]
        qkv = qkv.view(self.tokens, self.row)
        qkv.copy_(self.data)
        out = qkv if in_place else torch.full((self.tokens, self.heads * self.dim), 7.25, dtype=self.dtype, device="cuda:0")
        pools = [torch.full((self.num_pages, self.page_bytes), 0xa5, dtype=torch.uint8, device="cuda:0") for _ in range(2)]
        up = lambda a: torch.from_numpy(a).cuda()  # noqa: E731
        kept = up(self.freq), up(self.positions), up(self.slots)
        size, h, g = self.dim * 2, self.heads, self.kv_heads
        at = qkv.data_ptr()
        native.call("kudacuda_rope_paged_append_mx", at, at + h * size, at + (h + g) * size, *[x.data_ptr() for x in kept],
                    out.data_ptr(), pools[0].data_ptr(), pools[1].data_ptr(), CODE[self.dtype], self.bits, self.tokens, h, g,
                    self.dim, self.rotary, int(self.pairs), self.row, self.row, self.row, out.stride(0), self.num_pages,
                    self.page, self.page_bytes, self.amplitude, torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        return f64(out[:, :h * self.dim]).reshape(self.tokens, h, self.dim), [p.cpu().numpy() for p in pools]

    def want(self):
        """The pools' bytes: where two 64-bit forms of a turn differ (by 2^-50) next to a border of the type's or the
        block's rounding, a byte could differ too -- one number in 2^40, and these inputs are fixed."""

        _, k, v = self.parts()
        turned = rope(k, self.positions, self.freq, self.amplitude, self.pairs)
        turned = torch.from_numpy(turned).float().to(self.dtype).double().numpy()
        pools = []
        for x in (turned, v):
            codes, blocks = mx.pack(x, self.bits, self.dtype)
            data = np.full((self.num_pages, self.page_bytes), 0xa5, dtype=np.uint8)
            row, n = self.dim * self.bits // 8, self.kv_heads * self.page
            elements = data[:, :n * row].reshape(-1, self.kv_heads, self.page, row)  # (copies: put back below)
            powers = data[:, n * row:n * (row + self.dim // 32)].reshape(-1, self.kv_heads, self.page, self.dim // 32)
            for i, slot in enumerate(self.slots):
                if 0 <= slot < self.num_pages * self.page:
                    elements[slot // self.page, :, slot % self.page] = mx.to_bytes(codes[i], self.bits)
                    powers[slot // self.page, :, slot % self.page] = blocks[i]
            data[:, :n * row] = elements.reshape(self.num_pages, -1)
            data[:, n * row:n * (row + self.dim // 32)] = powers.reshape(self.num_pages, -1)
            pools.append(data)
        return pools


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("kw", [
    dict(tokens=1), dict(tokens=8, heads=16, dim=128), dict(tokens=37, dim=128, pairs=True, amplitude=1.1386),
    dict(tokens=50, rotary=32, kv_heads=1, heads=7), dict(tokens=19, dim=128, rotary=64, pairs=True, page=64, extra=32),
    dict(tokens=33, rotary=2), dict(tokens=33, rotary=6, pairs=True), dict(tokens=21, dim=128, rotary=30),
    dict(tokens=40, gap=3, offset=1), dict(tokens=40, dim=128, gap=5, pairs=True), dict(tokens=2050, heads=2, kv_heads=1),
    dict(tokens=2049, heads=3, kv_heads=3, gap=1, rotary=16), dict(tokens=30, kv_heads=8, heads=8, page=256),
    dict(tokens=10, padding=((0, -1), (3, 1 << 40), (9, 3 * 16 + 16))),
], ids=str)
def test_append_writes_the_bytes_of_the_definition(torch_gpu, native, dtype, bits, kw):
    case = Append(5, bits=bits, dtype=dtype, **kw)
    print(f"append {kw} {bits} bits {dtype}", flush=True)
    queries, pools = case.call(native)
    for got, want in zip(pools, case.want()):
        assert np.array_equal(got, want)
    q = case.parts()[0]
    want = rope(q, case.positions, case.freq, case.amplitude, case.pairs)
    off = np.abs(queries - want)
    live = (case.slots >= 0) & (case.slots < case.num_pages * case.page)
    assert (off <= rope_bound(q, want, case.rotary // 2, case.pairs, case.amplitude, dtype))[live].all()
    assert (queries[~live] == 7.25).all()
    in_place, again = case.call(native, in_place=True)
    assert np.array_equal(in_place[live], queries[live]) and all(np.array_equal(a, b) for a, b in zip(again, pools))


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("bits", [4, 8])
def test_every_number_of_the_type(torch_gpu, native, dtype, bits):
    """All 2^16 patterns as values: neighbours in a block, and mixed ones."""

    patterns = np.arange(65536, dtype=np.uint16)
    mixed = np.random.default_rng(1).permutation(patterns)
    x = torch.from_numpy(np.concatenate([patterns, mixed]).view(np.int16)).view(dtype).view(-1, 2, 64)
    case = Append(6, x.shape[0], heads=2, kv_heads=2, bits=bits, dtype=dtype)
    case.qkv[:, 4 * 64:] = x.flatten(1)
    case.data[:, 4 * 64:] = x.flatten(1)
    with np.errstate(invalid="ignore"):
        want = case.want()
    assert np.array_equal(case.call(native)[1][1], want[1])


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("bits", [4, 8])
def test_sizes_on_the_border_of_two_exponents(torch_gpu, native, dtype, bits):
    """A largest magnitude at and next to 7 (464) times a power of two, and elements half way between two levels."""

    levels = np.unique(np.abs(mx.levels(bits)[np.isfinite(mx.levels(bits))]))
    half = (levels[1:] + levels[:-1]) / 2
    rows = []
    for power in (-6, -1, 0, 3, 7):
        for top in (7.0, 6.0) if bits == 4 else (464.0, 448.0):
            for step in (-1, 0, 1):
                top16 = torch.tensor(top * 2.0**power if bits == 4 else top * 2.0 ** (power - 6)).to(dtype).view(torch.int16)
                value = (top16 + step).view(dtype).double().item()
                m = np.resize(np.concatenate([half, -half, levels]), 32 * -(-3 * len(half) // 32)) * (value / top)
                for block in m.reshape(-1, 32):
                    rows.append(np.concatenate([[value], block[1:], [-value], block[:31]]))
    x = torch.from_numpy(np.array(rows)).to(dtype)
    case = Append(7, len(rows), heads=1, kv_heads=1, bits=bits, dtype=dtype)
    case.qkv[:, 128:] = x
    case.data[:, 128:] = x
    assert np.array_equal(case.call(native)[1][1], case.want()[1])


def _read(native, pools, slots, dtype, bits, kv_heads, dim, page, gap=0):
    out = [torch.full((len(slots), kv_heads * dim + gap), 7.25, dtype=dtype, device="cuda:0") for _ in range(2)]
    slots = torch.from_numpy(slots).cuda()
    native.call("kudacuda_paged_read_mx", pools[0].data_ptr(), pools[1].data_ptr(), slots.data_ptr(), out[0].data_ptr(),
                out[1].data_ptr(), CODE[dtype], bits, len(slots), kv_heads, dim, out[0].stride(0), out[1].stride(0),
                pools[0].shape[0], page, pools[0].stride(0), torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    return [f64(x) for x in out]


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("tokens,kv_heads,dim,page,extra,gap", [
    (1, 1, 64, 16, 0, 0), (300, 2, 128, 16, 0, 8), (77, 7, 64, 256, 48, 0), (5000, 1, 128, 64, 16, 0), (40000, 4, 64, 16, 0, 0)])
def test_read_gives_every_code_and_power(torch_gpu, native, dtype, bits, tokens, kv_heads, dim, page, extra, gap):
    rng = np.random.default_rng([tokens, dim])
    pages = -(-tokens // page) + 2
    low, high = mx.exponents(bits, dtype)
    pools, values = [], []
    for _ in range(2):
        codes = rng.integers(0, 1 << bits, (pages, kv_heads, page, dim), dtype=np.uint8)
        blocks = rng.integers(low + 127, high + 128, (pages, kv_heads, page, dim // 32)).astype(np.uint8)
        blocks[rng.random(blocks.shape) < 0.02] = 255
        pools.append(torch.from_numpy(mx.to_pages(codes, blocks, bits, extra)).cuda())
        values.append(mx.unpack(codes, blocks, bits))
    slots = rng.integers(0, pages * page, tokens).astype(np.int64)
    if tokens > 10:
        slots[[3, 7]] = -1, pages * page
    live = (slots >= 0) & (slots < pages * page)
    at = np.where(live, slots, 0)
    for got, want in zip(_read(native, pools, slots, dtype, bits, kv_heads, dim, page, gap), values):
        want = want[at // page, :, at % page].reshape(tokens, -1)
        assert np.array_equal(got[live, :kv_heads * dim], want[live], equal_nan=True)
        assert (got[~live] == 7.25).all() and (got[:, kv_heads * dim:] == 7.25).all()


def test_pages_past_32_bits(torch_gpu, native):
    """Pages 2^26 bytes apart in pools that overlap: rows beyond 4 GB come back, and nothing before them changes."""

    stride, pages, bits, dim = 1 << 26, 70, 4, 64
    pool = torch.zeros(pages * stride, dtype=torch.uint8, device="cuda:0")
    case = Append(8, 40, bits=bits)
    case.num_pages = 3
    slots = case.slots % 48
    case.slots = np.unique(slots)[:30]
    n = len(case.slots)
    qkv = case.data[:n].cuda()
    out = torch.empty((n, 4 * dim), dtype=BF16, device="cuda:0")
    far = case.slots + (pages - 3) * 16
    up = lambda a: torch.from_numpy(a).cuda()  # noqa: E731
    kept = up(case.freq), up(case.positions[:n].copy()), up(far)
    keys, values = pool.data_ptr(), pool.data_ptr() + stride // 2
    native.call("kudacuda_rope_paged_append_mx", qkv.data_ptr(), qkv.data_ptr() + 4 * dim * 2, qkv.data_ptr() + 6 * dim * 2,
                *[x.data_ptr() for x in kept], out.data_ptr(), keys, values, 1, bits, n, 4, 2, dim, dim, 0, case.row, case.row,
                case.row, 4 * dim, pages, 16, stride, 1.0, torch.cuda.current_stream().cuda_stream)
    rows = torch.empty((2, n, 2, dim), dtype=BF16, device="cuda:0")
    native.call("kudacuda_paged_read_mx", keys, values, kept[2].data_ptr(), rows[0].data_ptr(), rows[1].data_ptr(), 1, bits, n, 2,
                dim, 2 * dim, 2 * dim, pages, 16, stride, torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    _, _, v = case.parts()
    codes, blocks = mx.pack(v[:n], bits, BF16)
    assert np.array_equal(f64(rows[1]), mx.unpack(codes, blocks, bits))
    assert int(pool[:(pages - 3) * stride].count_nonzero()) == 0
    del pool
    torch.cuda.empty_cache()


# ------------------------------------------------------------- the cache's books
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_a_cache_reads_what_was_appended(torch_gpu, native, bits, dtype):
    """Forks, copies, truncation and compaction move rows as they are; attention works on what read gives."""

    cache = PagedKvCache(native, torch, layers=2, kv_heads=2, head_dim=64, num_pages=24, dtype=dtype, bits=bits)
    rng, truth = np.random.default_rng(4), {}
    freq = torch.zeros(32, dtype=torch.float64, device="cuda:0")  # no turn: rows are stored as they come

    def feed(sequences, counts):
        batch = cache.extend(sequences, counts)
        starts = batch.query_starts.cpu().numpy()
        for layer in range(2):
            k, v = (torch.from_numpy(rng.standard_normal((batch.tokens, 2, 64)).astype(np.float32)).to(dtype) for _ in range(2))
            q = torch.zeros((batch.tokens, 4, 64), dtype=dtype, device="cuda:0")
            cache.append(layer, batch, q, k.cuda(), v.cuda(), freq)
            for i, s in enumerate(sequences):
                rows = truth.setdefault(s, [[[], []] for _ in range(2)])[layer]
                for kept, x in zip(rows, (k, v)):
                    codes, blocks = mx.pack(f64(x[starts[i]:starts[i + 1]]), bits, dtype)
                    kept += list(mx.unpack(codes, blocks, bits))
        return batch

    def holds():
        for s, layers in truth.items():
            for layer, rows in enumerate(layers):
                for got, want in zip(cache.read(layer, s), rows):
                    assert np.array_equal(f64(got), np.array(want)), (s, layer)

    a, b = cache.create(), cache.create()
    feed([a, b], [21, 16])
    c, d = cache.fork(a), cache.fork(a)
    for s in (c, d):
        truth[s] = [[list(r) for r in layer] for layer in truth[a]]
    feed([a, c, d], [1, 2, 4])
    holds()
    feed([b], [40])
    cache.free(a)
    truth.pop(a)
    cache.truncate(b, 33)
    truth[b] = [[r[:33] for r in layer] for layer in truth[b]]
    assert cache.compact() > 0
    holds()
    batch = feed([b, c, d], [9, 1, 20])
    holds()
    keys, values = cache.read(1, d, 5, 30)
    assert np.array_equal(f64(keys), np.array(truth[d][1][0][5:30])) and values.shape == (25, 2, 64)
    assert cache.read(0, c, 3, 3)[0].shape == (0, 2, 64)
    # a 16-bit cache with the same rows attends alike
    plain = PagedKvCache(native, torch, layers=1, kv_heads=2, head_dim=64, num_pages=24, dtype=dtype)
    q = torch.from_numpy(rng.standard_normal((batch.tokens, 4, 64)).astype(np.float32)).to(dtype).cuda()
    got = cache.attend(1, batch, q)
    ids = [plain.create() for _ in range(3)]
    old = [cache.length(s) - n for s, n in zip((b, c, d), (9, 1, 20))]
    for counts, part in ((old, lambda s, n: slice(0, n)), ((9, 1, 20), lambda s, n: slice(cache.length(s) - n, None))):
        mine = plain.extend(ids, counts)
        rows = [cache.read(1, s) for s in (b, c, d)]
        k, v = (torch.cat([r[j][part(s, n)] for r, s, n in zip(rows, (b, c, d), counts)]) for j in range(2))
        plain.append(0, mine, torch.zeros((mine.tokens, 4, 64), dtype=dtype, device="cuda:0"), k, v, freq)
    want = plain.attend(0, mine, q)
    # the same numbers through the same sums in another order: each is off by half a step of its own, and of its weights
    # (sum |weight * value| <= the largest value)
    most = max(float(np.abs(np.array(truth[x][1][1])).max()) for x in (b, c, d))
    assert (np.abs(f64(got) - f64(want)) <= 2 * (HALF[dtype] * np.abs(f64(want)) + (HALF[dtype] + 2.0**-11) * most)).all()
    assert np.array_equal(f64(plain.read(0, ids[0])[0]), np.array(truth[b][1][0]))
