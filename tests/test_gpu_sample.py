"""GPU: sampling (kudacuda_sample_tokens) against its definition in 64 bits.

Weights are rounded to 2^-42 of the largest and exp is off by a few 2^-52, so a cumulative sum over n tokens is off by
less than n 2^-43 + 2^-48 of the largest weight: tokens are compared where u (and top_p) is further than 2^-22 of the
sum (n <= 2^20) from the place where another token comes out, which leaves out next to none."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from tests._paged_ref import CODE, sample

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _call(native, logits, u, temperature=None, top_k=None, top_p=None, min_p=None, stream=None, chances=True,
          workspace=None, out=None):
    rows, vocab = logits.shape
    nbytes = native.lib.kudacuda_sample_workspace_bytes(rows, vocab)
    if workspace is None:  # whatever it holds before
        workspace = torch.full((nbytes,), 255, dtype=torch.uint8, device="cuda:0")
    tokens = torch.full((rows,), -5, dtype=torch.int32, device="cuda:0") if out is None else out[0]
    chance = torch.full((rows,), -5.0, device="cuda:0") if out is None else out[1]
    up = lambda a, t: None if a is None else torch.from_numpy(np.ascontiguousarray(a, dtype=t)).cuda()  # noqa: E731
    settings = [a if torch.is_tensor(a) else up(a, t) for a, t in
                ((u, np.float32), (temperature, np.float32), (top_k, np.int32), (top_p, np.float32), (min_p, np.float32))]
    stream = torch.cuda.current_stream() if stream is None else stream
    torch.cuda.synchronize()
    native.call("kudacuda_sample_tokens", logits.data_ptr(), *[0 if a is None else a.data_ptr() for a in settings],
                tokens.data_ptr(), chance.data_ptr() if chances else 0, workspace.data_ptr(), nbytes,
                CODE[logits.dtype], rows, vocab, logits.stride(0), stream.cuda_stream)
    torch.cuda.synchronize()
    return tokens.cpu().numpy(), chance.cpu().numpy()


def _check(logits, got, u, temperature=None, top_k=None, top_p=None, min_p=None, least=0.9):
    """Every row whose draw is not next to a border; at least the share ``least`` of them."""

    tokens, chances = got
    x = logits.float().cpu().numpy()
    rows, clear = len(x), 0
    at = lambda a, i, off: off if a is None else a[i]  # noqa: E731
    for i in range(rows):
        token, chance, distance = sample(x[i], float(np.float32(u[i])), float(np.float32(at(temperature, i, 1.0))),
                                         int(at(top_k, i, 0)), float(np.float32(at(top_p, i, 1.0))),
                                         float(np.float32(at(min_p, i, 0.0))))
        if distance > 2.0**-22:
            clear += 1
            assert tokens[i] == token, (i, tokens[i], token)
            # the chance is rounded to fp32 once, its weight to 2^-42 and the sum as above
            assert abs(chances[i] - chance) <= 2.0**-23 * chance + 2.0**-40, (i, chances[i], chance)
    assert clear >= least * rows


def _logits(rng, rows, vocab, dtype, std=2.5, pitch=None, shift=0):
    pitch = vocab if pitch is None else pitch
    flat = torch.from_numpy((rng.standard_normal(rows * pitch + shift) * std).astype(np.float32)).to(dtype).cuda()
    return torch.as_strided(flat, (rows, vocab), (pitch, 1), shift)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab,pitch,shift", [
    (1, 1, None, 0), (3, 2, None, 0), (5, 7, 9, 1), (4, 2047, None, 0), (4, 2048, 2056, 0), (3, 2049, 2051, 3),
    (6, 32000, None, 0), (2, 151936, None, 0), (40, 5000, 5008, 8), (2, 1 << 20, None, 0), (2000, 33, None, 0),
    (63, 4100, None, 0), (64, 9000, None, 0), (300, 5000, 5003, 3),
])
def test_settings_row_by_row(torch_gpu, native, dtype, rows, vocab, pitch, shift):
    """Every row its own mix of settings, off and degenerate ones among them."""

    rng = np.random.default_rng([rows, vocab])
    logits = _logits(rng, rows, vocab, dtype, pitch=pitch, shift=shift)
    for _ in range(3):
        settings = dict(temperature=rng.choice([0.0, -1.0, 0.1, 0.7, 1.0, 1.5], rows),
                        top_k=rng.choice([-1, 0, 1, 2, 50, 900, 5000, 3 * vocab], rows),
                        top_p=rng.choice([-1.0, 0.0, 1e-6, 0.3, 0.9, 0.999, 1.0, 2.0], rows),
                        min_p=rng.choice([-1.0, 0.0, 1e-7, 0.05, 0.5, 1.0, 3.0], rows))
        u = rng.random(rows).astype(np.float32)
        u[0] = 0.0
        u[-1] = np.float32(1.0 - 2.0**-24)
        _check(logits, _call(native, logits, u, **settings), u, **settings, least=0.0 if rows < 10 else 0.85)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("name", ["temperature", "top_k", "top_p", "min_p", None])
def test_one_setting_alone(torch_gpu, native, dtype, name):
    rng = np.random.default_rng(3)
    rows, vocab = 12, 9000
    logits = _logits(rng, rows, vocab, dtype)
    u = rng.random(rows).astype(np.float32)
    values = {"temperature": 0.6, "top_k": 40, "top_p": 0.92, "min_p": 0.02}
    settings = {} if name is None else {name: np.full(rows, values[name])}
    _check(logits, _call(native, logits, u, **settings), u, **settings)


@pytest.mark.parametrize("dtype", TYPES)
def test_flat_rows_take_the_whole_row(torch_gpu, native, dtype):
    """More tokens in the deciding bucket than its list holds: equal logits (ties by id), and a high temperature."""

    rng = np.random.default_rng(8)
    rows, vocab = 10, 20000
    logits = _logits(rng, rows, vocab, dtype, std=1.0)
    logits[:4] = 1.5
    logits[4:6, ::3] = float("-inf")
    settings = dict(temperature=np.where(np.arange(rows) < 4, 1.0, 60.0),
                    top_k=np.array([5000, 0, 7000, 0, 0, 9000, 0, 12345, 3, 15000]),
                    top_p=np.array([1.0, 0.5, 0.25, 1.0, 0.7, 0.6, 0.9, 1.0, 0.5, 0.01]))
    for _ in range(3):
        u = rng.random(rows).astype(np.float32)
        # equal weights: the sums are whole numbers on both sides, borders included
        _check(logits, _call(native, logits, u, **settings), u, **settings, least=0.5)
    tokens, _ = _call(native, logits, np.full(rows, 1.0 - 2.0**-24), **settings)
    assert tokens[0] == 4999 and tokens[1] == 9999 and tokens[2] == 1749 and tokens[3] == 19999


def test_ties_go_to_the_lowest_ids(torch_gpu, native):
    logits = torch.full((4, 3000), -3.0, device="cuda:0")
    logits[:, 100:2900:7] = 2.0
    logits[2, 5] = float("nan")
    logits[:, 50], logits[:, 51] = -0.0, 0.0
    ids = np.arange(100, 2900, 7)
    top = 1.0 - 2.0**-24
    tokens, chances = _call(native, logits, [0.0, top, top, 0.5], temperature=[0.0, 0.01, 0.01, 0.01], top_k=[0, 3, 0, 1],
                            top_p=[1.0, 1.0, 0.1, 1.0])
    # 0.1 in fp32 is above 0.1: 40 of 400 equal weights do not reach it
    assert list(tokens) == [ids[0], ids[2], ids[40], ids[0]]
    assert np.array_equal(chances, np.float32([1.0, 1 / 3, 1 / 41, 1.0]))


def test_infinite_and_missing_logits(torch_gpu, native):
    inf, nan = float("inf"), float("nan")
    rows = torch.tensor([[1.0, inf, 0.0, inf], [nan, -inf, nan, -inf], [nan, -1.0, -inf, -1.0], [-inf, -inf, 2.0, nan],
                         [-3.0e38, 3.0e38, 0.0, nan]], device="cuda:0")
    u = [0.6, 0.6, 0.6, 0.6, 0.6]
    for settings in ({}, dict(top_k=[3] * 5), dict(top_p=[0.9] * 5), dict(top_k=[3] * 5, top_p=[0.9] * 5, min_p=[0.1] * 5)):
        tokens, chances = _call(native, rows, u, **settings)
        assert list(tokens) == [3, 0, 3, 2, 1], settings
        assert np.array_equal(chances, np.float32([0.5, 0.0, 0.5, 1.0, 1.0])), settings
    tokens, chances = _call(native, rows, u, temperature=[0.0] * 5)
    assert list(tokens) == [1, 0, 1, 2, 1] and list(chances) == [1.0, 0.0, 1.0, 1.0, 1.0]
    # numbers outside [0, 1) fall on the first and the last kept token
    logits = torch.zeros((4, 10), device="cuda:0")
    tokens, _ = _call(native, logits, [-1.0, nan, 1.0, inf], top_k=[4] * 4)
    assert list(tokens) == [0, 0, 3, 3]


def test_draws_follow_the_distribution(torch_gpu, native):
    """One row of logits, a grid of numbers: each token comes out for its share of them."""

    rng = np.random.default_rng(12)
    vocab, n = 4000, 4096
    row = _logits(rng, 1, vocab, torch.float32)
    u = ((np.arange(n) + 0.5) / n).astype(np.float32)
    tokens, chances = _call(native, row.expand(n, vocab).contiguous(), u, temperature=np.full(n, 0.7), top_p=np.full(n, 0.8))
    x = row.cpu().numpy()[0].astype(np.float64) / float(np.float32(0.7))
    p = np.exp(x - x.max())
    order = np.argsort(-p, kind="stable")
    kept = order[:np.count_nonzero(np.cumsum(p[order]) - p[order] < float(np.float32(0.8)) * p.sum())]
    share = np.zeros(vocab)
    share[kept] = p[kept] / p[kept].sum()
    # a token's share of the grid is its chance to within one number
    assert np.abs(np.bincount(tokens, minlength=vocab) / n - share).max() <= 1.0 / n + 1e-9
    assert np.abs(chances - share[tokens]).max() <= 1e-6


@pytest.mark.parametrize("rows", [6, 70])
def test_captured_call_without_chances_on_another_stream(torch_gpu, native, rows):
    """Replays read new logits, numbers and settings; the workspace is not cleared between them."""

    rng = np.random.default_rng(14)
    vocab = 30000
    logits = _logits(rng, rows, vocab, torch.bfloat16)
    u, temperature, top_p, min_p = (torch.zeros(rows, device="cuda:0") for _ in range(4))
    top_k = torch.zeros(rows, dtype=torch.int32, device="cuda:0")
    tokens = torch.zeros(rows, dtype=torch.int32, device="cuda:0")
    nbytes = native.lib.kudacuda_sample_workspace_bytes(rows, vocab)
    workspace = torch.full((nbytes,), 1, dtype=torch.uint8, device="cuda:0")
    side = torch.cuda.Stream()
    args = (logits.data_ptr(), u.data_ptr(), temperature.data_ptr(), top_k.data_ptr(), top_p.data_ptr(), min_p.data_ptr(),
            tokens.data_ptr(), 0, workspace.data_ptr(), nbytes, 1, rows, vocab, vocab)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        native.call("kudacuda_sample_tokens", *args, torch.cuda.current_stream().cuda_stream)
    for _ in range(4):
        values = dict(temperature=rng.choice([0.0, 0.7, 1.2], rows), top_k=rng.choice([0, 20, 3000], rows),
                      top_p=rng.choice([0.5, 0.95, 1.0], rows), min_p=rng.choice([0.0, 0.01], rows))
        numbers = rng.random(rows).astype(np.float32)
        with torch.cuda.stream(side):
            logits.copy_(_logits(rng, rows, vocab, torch.bfloat16))
            u.copy_(torch.from_numpy(numbers))
            for t, name in ((temperature, "temperature"), (top_k, "top_k"), (top_p, "top_p"), (min_p, "min_p")):
                t.copy_(torch.from_numpy(np.asarray(values[name])))
            graph.replay()
        side.synchronize()
        eager, chances = _call(native, logits, numbers, **values)
        assert np.array_equal(tokens.cpu().numpy(), eager)
        _check(logits, (eager, chances), numbers, **values, least=0.6)


@pytest.mark.parametrize("rows", [1, 7, 64, 301])
@pytest.mark.parametrize("vocab", [1, 2049, 40000])
def test_calls_stay_inside_their_workspace(torch_gpu, native, rows, vocab):
    rng = np.random.default_rng([15, rows, vocab])
    logits = _logits(rng, rows, vocab, torch.float16, std=0.5)
    u = torch.from_numpy(rng.random(rows).astype(np.float32)).cuda()
    top_k = torch.from_numpy(rng.choice([0, 3, 500, 30000], rows).astype(np.int32)).cuda()
    top_p = torch.from_numpy(rng.choice([0.4, 0.97, 1.0], rows).astype(np.float32)).cuda()
    tokens = torch.full((rows + 1,), -5, dtype=torch.int32, device="cuda:0")
    nbytes = native.lib.kudacuda_sample_workspace_bytes(rows, vocab)
    workspace = torch.full((nbytes + 4096,), 0x7f, dtype=torch.uint8, device="cuda:0")
    native.call("kudacuda_sample_tokens", logits.data_ptr(), u.data_ptr(), 0, top_k.data_ptr(), top_p.data_ptr(), 0,
                tokens.data_ptr(), 0, workspace.data_ptr(), nbytes, 2, rows, vocab, vocab,
                torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert (workspace[nbytes:] == 0x7f).all()
    assert (tokens[:-1] >= 0).all() and (tokens[:-1] < vocab).all() and int(tokens[-1]) == -5
