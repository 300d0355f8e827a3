"""GPU: the paged-cache operators as a server runs them, round after round, against the one-sequence decoder.

A two-layer Qwen2.5-3B-shaped NF4 model (Qwen2Nf4Decoder's own weights) serves three sequences from one paged cache:
projections by the multi-token GEMMs, rotary append, chunk attention, sampling.  Prompts enter in chunks while other
sequences decode, one sequence is forked and one leaves, the cache is compacted in between."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from kudacuda_amd import synthetic
from kudacuda_amd.paged_cache import OutOfPages, PagedKvCache
from kudacuda_amd.qwen2_decoder import Qwen2Nf4Decoder
from kudacuda_amd.rotary import rope_frequencies
from tests._paged_ref import sample

pytestmark = pytest.mark.gpu
SEED, LAYERS, VOCAB = 20261207, 2, 4096
HIDDEN, INTER, HEADS, KV_HEADS, DIM = 2048, 11008, 16, 2, 128


@pytest.fixture(scope="module")
def model(torch_gpu, native):
    gpu = Qwen2Nf4Decoder.synthetic(native, torch_gpu, seed=SEED, num_layers=LAYERS, vocab=VOCAB, kv_capacity=256,
                                    token_capacity=256)
    yield gpu
    gpu.close()


class Server:
    """The forward pass of a batch of new tokens; everything on torch's current stream."""

    def __init__(self, native, model, num_pages=64, page_size=16):
        self.native, self.model = native, model
        self.cache = PagedKvCache(native, torch, layers=LAYERS, kv_heads=KV_HEADS, head_dim=DIM, num_pages=num_pages,
                                  page_size=page_size)
        self.freq = torch.from_numpy(rope_frequencies(DIM, model.cfg.rope_theta)[0]).cuda()

    def _norm(self, x, gamma):
        y = x.float()
        return (y * torch.rsqrt(y.pow(2).mean(dim=1, keepdim=True) + self.model.cfg.eps) * gamma.float()).bfloat16()

    def _gemm(self, x, layer, name, n, k, bias=None, residual=None, out=None):
        out = torch.empty((x.shape[0], n), dtype=torch.bfloat16, device="cuda:0") if out is None else out
        self.native.call("kudacuda_nf4_gemm_bf16", x.data_ptr(), layer[f"{name}_packed"].data_ptr(),
                         layer[f"{name}_absmax"].data_ptr(), 0 if bias is None else bias.data_ptr(),
                         0 if residual is None else residual.data_ptr(), out.data_ptr(), x.shape[0], k, n, 64,
                         torch.cuda.current_stream().cuda_stream)
        return out

    def forward(self, sequences, tokens):
        """Logits [sequences, vocab] after each sequence's last new token."""

        batch = self.cache.extend(sequences, [len(t) for t in tokens])
        ids = torch.from_numpy(np.concatenate(tokens).astype(np.int64)).cuda()
        x = self.model.embed[ids]
        for li, layer in enumerate(self.model.layers):
            h = self._norm(x, layer["input_norm"])
            q = self._gemm(h, layer, "q", HIDDEN, HIDDEN, layer["q_bias"]).view(-1, HEADS, DIM)
            k, v = (self._gemm(h, layer, n, KV_HEADS * DIM, HIDDEN, layer[f"{n}_bias"]).view(-1, KV_HEADS, DIM)
                    for n in ("k", "v"))
            q = self.cache.append(li, batch, q, k, v, self.freq, out=q)
            a = self.cache.attend(li, batch, q)
            x = self._gemm(a.view(-1, HIDDEN), layer, "o", HIDDEN, HIDDEN, residual=x)
            h = self._norm(x, layer["post_norm"])
            m = torch.empty((h.shape[0], INTER), dtype=torch.bfloat16, device="cuda:0")
            self.native.call("kudacuda_nf4_gemm_swiglu_bf16", h.data_ptr(), layer["gate_packed"].data_ptr(),
                             layer["gate_absmax"].data_ptr(), layer["up_packed"].data_ptr(),
                             layer["up_absmax"].data_ptr(), m.data_ptr(), h.shape[0], HIDDEN, INTER, 64,
                             torch.cuda.current_stream().cuda_stream)
            x = self._gemm(m, layer, "down", HIDDEN, INTER, residual=x)
        last = x[(batch.query_starts[1:] - 1).long()].contiguous()
        logits = torch.empty((len(sequences), VOCAB), dtype=torch.bfloat16, device="cuda:0")
        greedy = torch.empty(len(sequences), dtype=torch.int32, device="cuda:0")
        for i in range(len(sequences)):
            self.native.call("kudacuda_lm_head_argmax_bf16", last[i].data_ptr(), self.model.final_norm.data_ptr(),
                             self.model.embed.data_ptr(), logits[i].data_ptr(), greedy[i:].data_ptr(), VOCAB, HIDDEN,
                             self.model.cfg.eps, torch.cuda.current_stream().cuda_stream)
        return logits, greedy

    def sample(self, logits, u, **settings):
        rows = logits.shape[0]
        up = lambda a, t: torch.from_numpy(np.asarray(a, dtype=t)).cuda()  # noqa: E731
        kept = [up(u, np.float32)] + [up(settings[n], t) if n in settings else None for n, t in
                                      (("temperature", np.float32), ("top_k", np.int32), ("top_p", np.float32),
                                       ("min_p", np.float32))]
        tokens = torch.empty(rows, dtype=torch.int32, device="cuda:0")
        chances = torch.empty(rows, device="cuda:0")
        nbytes = self.native.lib.kudacuda_sample_workspace_bytes(rows, VOCAB)
        workspace = torch.empty(nbytes, dtype=torch.uint8, device="cuda:0")
        self.native.call("kudacuda_sample_tokens", logits.data_ptr(), *[0 if a is None else a.data_ptr() for a in kept],
                         tokens.data_ptr(), chances.data_ptr(), workspace.data_ptr(), nbytes, 1, rows, VOCAB, VOCAB,
                         torch.cuda.current_stream().cuda_stream)
        return tokens.cpu().numpy(), chances.cpu().numpy()


def _reference(model, tokens):
    """The decoder's cache rows [layers][keys, values] and logits after ``tokens``, one sequence at a time."""

    model.reset(np.asarray(tokens, dtype=np.int32))
    model.run_steps(len(tokens), graph=False)
    model.stream.synchronize()
    rows = [[layer[n][:, :len(tokens)].float().clone() for n in ("key_cache", "value_cache")] for layer in model.layers]
    return rows, model.logits.float().clone()


def _near(got, want):
    # ten bf16 roundings a layer lie between the two (norm, projections, rotation, attention, residuals, products),
    # each off by at most 2^-8 of its value: 20 * 2^-8 < 2^-3.6 at the worst, all in one direction
    assert float((got - want).norm()) <= 20 * 2.0**-8 * float(want.norm())


def _check_sequence(server, model, s, tokens, logits=None):
    rows, want = _reference(model, tokens)
    pages, n = server.cache.pages(s), server.cache.length(s)
    assert n == len(tokens)
    for li in range(LAYERS):
        for pool, ref in zip((server.cache.keys(li), server.cache.values(li)), rows[li]):
            _near(pool[pages].transpose(0, 1).flatten(1, 2)[:, :n].float(), ref)
    if logits is not None:
        _near(logits.float(), want)


@pytest.mark.parametrize("page_size", [16, 1])
def test_rounds_of_a_server_follow_the_decoder(torch_gpu, native, model, page_size):
    server = Server(native, model, num_pages=320 // page_size + 8, page_size=page_size)
    cache, rng = server.cache, np.random.default_rng(SEED)
    texts = {name: list(synthetic.prompt_ids(SEED + i, n, VOCAB)) for i, (name, n) in enumerate((("a", 50), ("b", 7), ("c", 33)))}
    ids = {name: cache.create() for name in texts}
    told = {name: [] for name in texts}

    def round_(feed):
        """One round: {sequence: new tokens}; returns {sequence: logits}."""

        names = list(feed)
        logits, greedy = server.forward([ids[n] for n in names], [feed[n] for n in names])
        for n in names:
            told[n] = told[n] + list(feed[n])
        tokens, chances = server.sample(logits, np.zeros(len(names)), temperature=np.zeros(len(names)))
        assert np.array_equal(tokens, greedy.cpu().numpy()) and (chances == 1.0).all()
        return dict(zip(names, logits))

    # prompts in chunks, short ones next to them
    round_({"a": texts["a"][:20], "b": texts["b"]})
    round_({"a": texts["a"][20:], "b": [17], "c": texts["c"][:1]})
    logits = round_({"c": texts["c"][1:], "b": [99], "a": [5]})
    for name in logits:
        _check_sequence(server, model, ids[name], told[name], logits[name])
    # a fork goes on by itself, its parent too
    ids["d"], told["d"] = cache.fork(ids["a"]), list(told["a"])
    logits = round_({"d": [1, 2, 3], "a": [4], "b": [6]})
    cache.free(ids.pop("b"))
    assert cache.compact() > 0
    logits = round_({"a": [7], "d": [8], "c": [9, 10]})
    for name in logits:
        _check_sequence(server, model, ids[name], told[name], logits[name])
    # sampled tokens on these logits
    batch = torch.stack([logits[n] for n in logits])
    settings = dict(temperature=[0.7, 1.0, 1.3], top_k=[0, 40, 500], top_p=[0.9, 0.95, 1.0], min_p=[0.0, 0.01, 0.0])
    for _ in range(5):
        u = rng.random(3).astype(np.float32)
        tokens, chances = server.sample(batch, u, **settings)
        x = batch.float().cpu().numpy()
        for i in range(3):
            token, chance, distance = sample(x[i], float(u[i]), *[float(np.float32(settings[n][i])) if n != "top_k" else
                                                                  settings[n][i] for n in ("temperature", "top_k", "top_p",
                                                                                           "min_p")])
            if distance > 2.0**-22:
                assert tokens[i] == token and abs(chances[i] - chance) <= 2.0**-23 * chance + 2.0**-40
    with pytest.raises(OutOfPages):
        server.forward([ids["a"]], [np.zeros(400, dtype=np.int64)])
    _check_sequence(server, model, ids["a"], told["a"])


def test_a_chunked_prompt_on_another_stream_equals_one_piece(torch_gpu, native, model):
    """The cache's own workspace and tables on a side stream: chunk by chunk or at once, the same rows and logits."""

    prompt = synthetic.prompt_ids(SEED + 9, 200, VOCAB)
    whole = Server(native, model)
    s = whole.cache.create()
    logits, _ = whole.forward([s], [prompt])
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        parts = Server(native, model)
        t = parts.cache.create()
        for at, end in ((0, 1), (1, 64), (64, 65), (65, 190), (190, 200)):
            piece, _ = parts.forward([t], [prompt[at:end]])
    side.synchronize()
    _near(piece.float(), logits.float())
    for li in range(LAYERS):
        for a, b in ((whole.cache.keys(li), parts.cache.keys(li)), (whole.cache.values(li), parts.cache.values(li))):
            _near(b[parts.cache.pages(t)].float(), a[whole.cache.pages(s)].float())
