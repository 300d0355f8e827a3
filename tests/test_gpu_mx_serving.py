"""GPU: a server's rounds over a cache of 8 or 4 bits, its requests with adapters of their own.

The two-layer NF4 model of the other serving tests: shared projections, adapters beside three of them, rotary append into
microscaled pages, attention over them; prompts in chunks next to single tokens, a fork, a sequence that leaves, compaction.
Each operator's outputs are compared with 64 bits on the inputs that it had there; the rows that the cache has to hold are
kept on the host, round after round."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from kudacuda_amd import synthetic
from kudacuda_amd.lora import LoraAdapters, lora_batch
from kudacuda_amd.paged_cache import PagedKvCache
from tests import _mx_ref as mx
from tests._paged_ref import HALF, f64, rope, rope_bound
from tests.test_gpu_serving import DIM, HEADS, HIDDEN, INTER, KV_HEADS, LAYERS, SEED, VOCAB, Server, model  # noqa: F401

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
PLACES = {"q": (HIDDEN, HEADS * DIM), "v": (HIDDEN, KV_HEADS * DIM), "down": (INTER, HIDDEN)}
RANKS = (16, 40, 3)


class MxServer(Server):
    """Rounds of requests, each of which names its adapter; every operator is followed in 64 bits."""

    def __init__(self, native, model, bits, num_pages=64, page_size=16):
        super().__init__(native, model, num_pages=1)
        self.cache = PagedKvCache(native, torch, layers=LAYERS, kv_heads=KV_HEADS, head_dim=DIM, num_pages=num_pages,
                                  page_size=page_size, bits=bits)
        self.bits, self.truth, self.checked = bits, {}, True
        rng = np.random.default_rng([SEED, bits])
        normal = lambda *s: torch.from_numpy(rng.standard_normal(s).astype(np.float32)).to(BF16)  # noqa: E731
        self.adapters, self.factors = {}, {}
        for li in range(LAYERS):
            for name, (inner, outer) in PLACES.items():
                pool = LoraAdapters(native, torch, in_features=inner, out_features=outer, adapters=len(RANKS), max_rank=64)
                for i, rank in enumerate(RANKS):
                    factors = normal(rank, inner) * inner**-0.5, normal(outer, rank) * 0.2
                    pool.load(i, *factors, scale=0.5)
                    self.factors[li, name, i] = [f64(f) for f in factors]
                self.adapters[li, name] = pool

    def adapt(self, li, name, plan, of, x, y):
        if not self.checked:
            return self.adapters[li, name].add(plan, x, y)
        base = f64(y)
        self.adapters[li, name].add(plan, x, y)
        want, bound, rows = base.copy(), np.zeros_like(base), f64(x)
        for i, adapter in enumerate(of):
            if adapter is not None:
                # the sums and parts of the adapters' own tests: in / 128 + 68 fp32 roundings of sum |x a|, a first
                # product in 17 bits of its row's largest, up to 256 more roundings behind it
                a, b = self.factors[li, name, adapter]
                u = a @ rows[i]
                want[i] += 0.5 * b @ u
                off = (x.shape[1] / 128 + 68) * 2.0**-24 * (np.abs(a) @ np.abs(rows[i]))
                bound[i] = 0.5 * np.abs(b) @ (off + (2.0**-17 + 2.0**-16) * np.abs(u).max())
        bound += HALF[BF16] * np.abs(want) + 2.0**-23 * np.abs(base) + 2.0**-25
        off = np.abs(f64(y) - want)
        assert (off <= bound).all(), (li, name, float((off / bound).max()))
        return y

    def append(self, li, batch, q, k, v):
        if not self.checked:
            return self.cache.append(li, batch, q, k, v, self.freq)
        inputs = [f64(x) for x in (q, k, v)]
        turned = self.cache.append(li, batch, q, k, v, self.freq)
        at, freq = batch.positions.cpu().numpy(), self.freq.cpu().numpy()
        want = rope(inputs[0], at, freq, 1.0, False)
        assert (np.abs(f64(turned) - want) <= rope_bound(inputs[0], want, DIM // 2, False, 1.0, BF16)).all()
        # (keys are formed in 64 bits: a code differs where two such forms, 2^-50 apart, lie on both sides of a border)
        key = torch.from_numpy(rope(inputs[1], at, freq, 1.0, False)).float().to(BF16).double().numpy()
        starts = batch.query_starts.cpu().numpy()
        for i, s in enumerate(batch.sequences):
            for kept, x in zip(self.truth.setdefault(s, [[[], []] for _ in range(LAYERS)])[li], (key, inputs[2])):
                kept += list(mx.unpack(*mx.pack(x[starts[i]:starts[i + 1]], self.bits, BF16), self.bits))
        return turned

    def attend(self, li, batch, q):
        out = self.cache.attend(li, batch, q)
        if not self.checked:
            return out
        got, queries = f64(out), f64(q)
        starts, scale = batch.query_starts.cpu().numpy(), float(np.float32(DIM**-0.5))
        for i, s in enumerate(batch.sequences):
            n = starts[i + 1] - starts[i]
            keys, values = (np.array(rows) for rows in self.truth[s][li])
            hidden = np.arange(len(keys))[None, :] > len(keys) - n + np.arange(n)[:, None]
            for h in range(HEADS):
                x, k, v = queries[starts[i]:starts[i + 1], h], keys[:, h * KV_HEADS // HEADS], values[:, h * KV_HEADS // HEADS]
                p = np.where(hidden, -np.inf, x @ k.T * scale)
                p = np.exp(p - p.max(axis=1, keepdims=True))
                p /= p.sum(axis=1, keepdims=True)
                want, size = p @ v, p @ np.abs(v)
                # a score is off by 128 roundings of sum |q k| in fp32 and by the query's parts, 2^-22 of the largest of a
                # block; a weight by that relatively, its sum again; and half a step for a weight's rounding and for the
                # sums of up to 2^11 of them
                tops = np.abs(x).reshape(n, -1, 32).max(axis=-1)
                blocks = np.abs(k).reshape(len(k), -1, 32).sum(axis=-1)
                off = scale * (2.0**-17 * (np.abs(x) @ np.abs(k).T) + 2.0**-22 * tops @ blocks.T)
                off = np.where(hidden, 0.0, off).max(axis=1, keepdims=True)
                assert off.max() < 0.1
                bound = HALF[BF16] * np.abs(want) + (HALF[BF16] + 2.2 * off + 2.0**-12) * size
                far = np.abs(got[starts[i]:starts[i + 1], h] - want)
                assert (far <= bound).all(), (li, s, h, float((far / bound).max()))
        return out

    def attention_block(self, li, layer, h, batch, plan, of):
        q = self._gemm(h, layer, "q", HIDDEN, HIDDEN, layer["q_bias"])
        k = self._gemm(h, layer, "k", KV_HEADS * DIM, HIDDEN, layer["k_bias"])
        v = self._gemm(h, layer, "v", KV_HEADS * DIM, HIDDEN, layer["v_bias"])
        q, v = self.adapt(li, "q", plan, of, h, q), self.adapt(li, "v", plan, of, h, v)
        q = self.append(li, batch, *(x.view(-1, x.shape[1] // DIM, DIM) for x in (q, k, v)))
        return self.attend(li, batch, q).view(-1, HIDDEN)

    def round(self, feed, names):
        """{sequence: new tokens}, {sequence: adapter}; the last layer's rows."""

        batch = self.cache.extend(list(feed), [len(t) for t in feed.values()])
        plan = lora_batch(torch, [names[s] for s in feed], [len(t) for t in feed.values()])
        of = [names[s] for s, t in feed.items() for _ in t]
        x = self.model.embed[torch.from_numpy(np.concatenate(list(feed.values())).astype(np.int64)).cuda()]
        for li, layer in enumerate(self.model.layers):
            a = self.attention_block(li, layer, self._norm(x, layer["input_norm"]), batch, plan, of)
            x = self._gemm(a, layer, "o", HIDDEN, HIDDEN, residual=x)
            h = self._norm(x, layer["post_norm"])
            m = torch.empty((h.shape[0], INTER), dtype=BF16, device="cuda:0")
            self.native.call("kudacuda_nf4_gemm_swiglu_bf16", h.data_ptr(), layer["gate_packed"].data_ptr(),
                             layer["gate_absmax"].data_ptr(), layer["up_packed"].data_ptr(), layer["up_absmax"].data_ptr(),
                             m.data_ptr(), h.shape[0], HIDDEN, INTER, 64, torch.cuda.current_stream().cuda_stream)
            x = self.adapt(li, "down", plan, of, m, self._gemm(m, layer, "down", HIDDEN, INTER, residual=x))
        return x

    def holds(self):
        for s, layers in self.truth.items():
            for li, rows in enumerate(layers):
                for got, want in zip(self.cache.read(li, s), rows):
                    assert np.array_equal(f64(got), np.array(want)), (s, li)


def _texts():
    return [list(synthetic.prompt_ids(SEED + i, n, VOCAB)) for i, n in enumerate((50, 7, 33))]


@pytest.mark.parametrize("bits,page_size", [(8, 16), (4, 16), (4, 64)])
def test_rounds_of_a_server_with_adapters(torch_gpu, native, model, bits, page_size):  # noqa: F811
    server = MxServer(native, model, bits, page_size=page_size)
    cache, texts = server.cache, _texts()
    a, b, c = (cache.create() for _ in range(3))
    names = {a: 0, b: None, c: 1}
    server.round({a: texts[0][:20], b: texts[1]}, names)
    server.round({b: [17], c: texts[2][:1], a: texts[0][20:]}, names)
    server.round({c: texts[2][1:], b: [99], a: [5]}, names)
    server.holds()
    # a fork goes on with another adapter, its parent too; one sequence leaves
    d = cache.fork(a)
    names[d] = 2
    server.truth[d] = [[list(r) for r in layer] for layer in server.truth[a]]
    server.round({d: [1, 2, 3], a: [4], b: [6]}, names)
    cache.free(b)
    server.truth.pop(b)
    cache.compact()
    server.holds()
    server.round({a: [7], d: [8], c: [9, 10]}, names)
    server.round({s: [s + 11] for s in (c, a, d)}, names)
    server.holds()


def test_rounds_on_another_stream_are_the_same(torch_gpu, native, model):  # noqa: F811
    """Rows, pages and adapters, everything on a side stream: the same bits."""

    def serve():
        server = MxServer(native, model, 4)
        server.checked = False
        a, b = server.cache.create(), server.cache.create()
        names = {a: 1, b: 0}
        out = [server.round(feed, names) for feed in ({a: _texts()[0]}, {a: [3], b: _texts()[2]}, {b: [4], a: [5]})]
        return out + [x for s in (a, b) for li in range(LAYERS) for x in server.cache.read(li, s)]

    want = serve()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        got = serve()
    side.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, want))


@pytest.mark.parametrize("bits", [8, 4])
def test_a_captured_round_replays(torch_gpu, native, model, bits):  # noqa: F811
    """Projections, adapters, append and attention of single tokens in a graph: every replay gives what the eager round
    gave, other inputs other results, with eager rounds between."""

    server = MxServer(native, model, bits)
    server.checked = False
    cache, layer = server.cache, model.layers[0]
    a, b = cache.create(), cache.create()
    names = {a: 0, b: 2}
    server.round({a: _texts()[0], b: _texts()[2]}, names)
    batch, plan = cache.extend([a, b], [1, 1]), lora_batch(torch, [0, 2], [1, 1])
    rows = torch.from_numpy(np.random.default_rng(bits).standard_normal((4, 2, HIDDEN)).astype(np.float32)).to(BF16).cuda()
    want = [server.attention_block(0, layer, x, batch, plan, [0, 2]).clone() for x in rows]
    h = rows[0].clone()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = server.attention_block(0, layer, h, batch, plan, [0, 2])
    other = cache.create()
    for i in (0, 1, 2, 3, 1, 0):
        h.copy_(rows[i])
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graph.replay()
        side.synchronize()
        assert torch.equal(out, want[i])
        server.round({other: [i]}, {other: 1})
        torch.cuda.synchronize()
    assert not torch.equal(want[0], want[1])
