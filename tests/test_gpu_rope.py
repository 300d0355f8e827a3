"""GPU: rotary positions (kudacuda_rope) and the append to a paged cache (kudacuda_rope_paged_append) against the
formula in 64 bits."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from kudacuda_amd.rotary import rope_frequencies
from tests._paged_ref import CODE, f64, rope, rope_bound

pytestmark = pytest.mark.gpu
SEED = 20261206


def _rows(rng, tokens, heads, dim, dtype, pitch=None, shift=0):
    """[tokens, heads, dim] on the GPU inside rows of ``pitch`` elements, ``shift`` elements behind their start."""

    pitch = heads * dim if pitch is None else pitch
    flat = torch.from_numpy(rng.standard_normal(tokens * pitch + shift).astype(np.float32)).to(dtype).cuda()
    return torch.as_strided(flat, (tokens, heads, dim), (pitch, dim, 1), shift)


def _turn(native, x, freq, positions, out, pairs, amplitude, stream=None):
    stream = torch.cuda.current_stream() if stream is None else stream
    native.call("kudacuda_rope", x.data_ptr(), freq.data_ptr(), positions.data_ptr(), out.data_ptr(), CODE[x.dtype],
                x.shape[0], x.shape[1], x.shape[2], 2 * freq.numel(), int(pairs), x.stride(0), out.stride(0), amplitude,
                stream.cuda_stream)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens,heads,dim,rotary,pairs,pitch,shift", [
    (1, 1, 128, 128, False, None, 0),
    (1, 16, 128, 128, True, None, 0),
    (5, 3, 64, 32, False, 3 * 64 + 8, 0),
    (5, 3, 64, 32, True, 3 * 64 + 8, 8),
    (7, 2, 128, 96, False, 2 * 128 + 1, 0),      # rows off 16-byte boundaries
    (7, 2, 80, 40, True, 160, 3),                # rotary dims that are no whole pieces, an odd beginning
    (3, 5, 2, 2, False, None, 0),
    (3, 1, 256, 254, True, None, 0),
    (2049, 2, 64, 64, False, None, 0),           # four tokens a block, one left over
    (2050, 1, 6, 4, True, 7, 0),
])
def test_rope_matches_fp64(torch_gpu, native, dtype, tokens, heads, dim, rotary, pairs, pitch, shift):
    rng = np.random.default_rng([SEED, tokens, dim, rotary])
    x = _rows(rng, tokens, heads, dim, dtype, pitch, shift)
    freq, amplitude = rope_frequencies(rotary, 1.0e4, scaling="yarn", factor=4.0, original_positions=4096)
    amplitude = float(np.float32(amplitude))
    positions = rng.integers(0, 1 << 20, tokens).astype(np.int32)
    positions[0] = 0 if tokens == 1 else 2**31 - 1
    d_freq, d_pos = torch.from_numpy(freq).cuda(), torch.from_numpy(positions).cuda()
    out = torch.full((tokens, heads, dim), 3.0, dtype=dtype, device="cuda:0")
    _turn(native, x, d_freq, d_pos, out, pairs, amplitude)
    want = rope(f64(x), positions, freq, amplitude, pairs)
    # far positions: the product position * frequency has 53 bits, 2^31 * 2^-53 < 2^-22 of an angle
    bound = rope_bound(f64(x), want, rotary // 2, pairs, amplitude, dtype)
    assert (np.abs(f64(out) - want) <= bound).all()
    assert torch.equal(out[..., rotary:], x[..., rotary:])
    # in place, and nothing between the rows
    before = torch.as_strided(x, (x.untyped_storage().nbytes() // 2,), (1,), 0).clone()
    _turn(native, x, d_freq, d_pos, x, pairs, amplitude)
    assert torch.equal(x, out)
    after = torch.as_strided(x, before.shape, (1,), 0)
    torch.as_strided(before, x.shape, x.stride(), shift).copy_(out)
    assert torch.equal(before, after)


def test_rope_of_negative_positions_turns_back(torch_gpu, native):
    rng = np.random.default_rng([SEED, 3])
    x = _rows(rng, 40, 2, 64, torch.float16)
    freq = torch.from_numpy(rope_frequencies(64)[0]).cuda()
    positions = torch.from_numpy(-rng.integers(0, 5000, 40).astype(np.int32)).cuda()
    out = torch.empty_like(x)
    _turn(native, x, freq, positions, out, False, 1.0)
    want = rope(f64(x), f64(positions), f64(freq), 1.0, False)
    assert (np.abs(f64(out) - want) <= rope_bound(f64(x), want, 32, False, 1.0, torch.float16)).all()


def _append(native, qkv, heads, kv_heads, dim, freq, positions, slots, out, keys, values, strides, page, pairs,
            amplitude, stream=None):
    stream = torch.cuda.current_stream() if stream is None else stream
    base, row = qkv.data_ptr(), qkv.stride(0)
    native.call("kudacuda_rope_paged_append", base, base + 2 * heads * dim, base + 2 * (heads + kv_heads) * dim,
                freq.data_ptr(), positions.data_ptr(), slots.data_ptr(), out.data_ptr(), keys.data_ptr(),
                values.data_ptr(), CODE[qkv.dtype], positions.numel(), heads, kv_heads, dim, 2 * freq.numel(),
                int(pairs), row, row, row, heads * dim, keys.shape[0], page, *strides, amplitude, stream.cuda_stream)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens,heads,kv_heads,dim,rotary,pairs,page,layout", [
    (1, 16, 2, 128, 128, False, 16, "hnd"),
    (37, 7, 1, 64, 64, True, 1, "hnd"),
    (37, 4, 4, 128, 64, False, 64, "nhd"),
    (50, 3, 3, 24, 10, True, 4, "nhd"),        # no whole pieces
    (2100, 8, 2, 64, 32, False, 16, "hnd"),
])
def test_append_fills_its_slots_and_nothing_else(torch_gpu, native, dtype, tokens, heads, kv_heads, dim, rotary, pairs,
                                                 page, layout):
    rng = np.random.default_rng([SEED, tokens, dim, page])
    qkv = _rows(rng, tokens, heads + 2 * kv_heads, dim, dtype)
    pages = -(-tokens // page) + 3
    slots = rng.permutation(pages * page)[:tokens].astype(np.int64)
    padding = rng.random(tokens) < (0.2 if tokens > 1 else 0.0)
    slots[padding] = rng.choice([-1, -2**40, pages * page, 2**50], padding.sum())
    positions = rng.integers(0, 200000, tokens).astype(np.int32)
    freq, amplitude = rope_frequencies(rotary, 1.0e6, scaling="linear", factor=2.0)
    shape = (pages, kv_heads, page, dim) if layout == "hnd" else (pages, page, kv_heads, dim)
    keys, values = (torch.full(shape, 9.0, dtype=dtype, device="cuda:0") for _ in range(2))
    strides = keys.stride()[:3] if layout == "hnd" else (keys.stride(0), keys.stride(2), keys.stride(1))
    out = torch.full((tokens, heads, dim), 9.0, dtype=dtype, device="cuda:0")
    _append(native, qkv, heads, kv_heads, dim, torch.from_numpy(freq).cuda(), torch.from_numpy(positions).cuda(),
            torch.from_numpy(slots).cuda(), out, keys, values, strides, page, pairs, amplitude)
    x = f64(qkv)
    turned = rope(x[:, :heads + kv_heads], positions, freq, amplitude, pairs)
    bound = rope_bound(x[:, :heads + kv_heads], turned, rotary // 2, pairs, amplitude, dtype)
    want_q, live = np.full((tokens, heads, dim), 9.0), ~padding
    want_q[live] = turned[live, :heads]
    assert (np.abs(f64(out) - want_q)[live] <= bound[live, :heads]).all()
    assert (f64(out)[padding] == 9.0).all()
    by_slot = [f64(p if layout == "nhd" else p.transpose(1, 2)).reshape(pages * page, kv_heads, dim)
               for p in (keys, values)]
    assert (np.abs(by_slot[0][slots[live]] - turned[live, heads:]) <= bound[live, heads:]).all()
    assert np.array_equal(by_slot[1][slots[live]], x[live, heads + kv_heads:])
    rest = np.ones(pages * page, dtype=bool)
    rest[slots[live]] = False
    assert (by_slot[0][rest] == 9.0).all() and (by_slot[1][rest] == 9.0).all()


def test_append_on_another_stream_and_in_a_captured_graph(torch_gpu, native):
    """Captured once, replayed with new rows, positions and slots, eager work in between."""

    rng = np.random.default_rng([SEED, 9])
    tokens, heads, kv_heads, dim, page, pages = 20, 4, 2, 64, 16, 6
    freq = torch.from_numpy(rope_frequencies(dim)[0]).cuda()
    qkv = _rows(rng, tokens, heads + 2 * kv_heads, dim, torch.bfloat16)
    positions = torch.zeros(tokens, dtype=torch.int32, device="cuda:0")
    slots = torch.full((tokens,), -1, dtype=torch.int64, device="cuda:0")
    out = torch.zeros((tokens, heads, dim), dtype=torch.bfloat16, device="cuda:0")
    keys, values = (torch.zeros((pages, kv_heads, page, dim), dtype=torch.bfloat16, device="cuda:0") for _ in range(2))
    args = (qkv, heads, kv_heads, dim, freq, positions, slots, out, keys, values, keys.stride()[:3], page, False, 1.0)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        _append(native, *args, stream=torch.cuda.current_stream())
    for round_ in range(3):
        with torch.cuda.stream(side):
            qkv.copy_(_rows(rng, tokens, heads + 2 * kv_heads, dim, torch.bfloat16))
            positions.copy_(torch.from_numpy(rng.integers(0, 9999, tokens).astype(np.int32)))
            slots.copy_(torch.from_numpy(rng.permutation(pages * page)[:tokens].astype(np.int64)))
            for t in (out, keys, values):
                t.zero_()
            graph.replay()
        side.synchronize()
        got = [t.clone() for t in (out, keys, values)]
        for t in (out, keys, values):
            t.zero_()
        torch.cuda.synchronize()
        _append(native, *args, stream=side)
        side.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, (out, keys, values))), round_
        assert bool((out != 0).any())


def test_no_tokens_is_a_call_that_does_nothing(torch_gpu, native):
    freq = torch.from_numpy(rope_frequencies(64)[0]).cuda()
    x = torch.full((1, 1, 64), 5.0, dtype=torch.bfloat16, device="cuda:0")
    positions = torch.zeros(1, dtype=torch.int32, device="cuda:0")
    native.call("kudacuda_rope", x.data_ptr(), freq.data_ptr(), positions.data_ptr(), x.data_ptr(), 1, 0, 1, 64, 64, 0,
                64, 64, 1.0, torch.cuda.current_stream().cuda_stream)
    assert (f64(x) == 5.0).all()
