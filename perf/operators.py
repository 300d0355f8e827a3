"""What serving several sequences from a paged KV cache takes, as cases that can be timed and compared.

A server keeps the rows of every sequence in pages of a fixed number of tokens
and does, round by round, four things that the one-sequence path does with its
one contiguous cache and its greedy argmax:

* ``rope`` -- rotate the new tokens' queries and keys and write keys and values
  into their pages (``kudacuda_rope_paged_append``);
* ``attention`` -- attend from the new tokens of every sequence, one token or a
  chunk of a prompt each, to all of that sequence's pages
  (``kudacuda_paged_attention``);
* ``pages`` -- copy pages inside the cache: the shared last page of a forked
  sequence, or all pages above a limit to free ones below it
  (``kudacuda_copy_pages``);
* ``sample`` -- draw the next token of every row of logits with temperature,
  top-k, top-p and min-p from one given random number a row, and tell the
  chance it had (``kudacuda_sample_tokens``).

With ``own`` false, ``run`` computes them in elementary torch operations, in 32
bits (angles, and everything a sampled token depends on, in 64).
"""

from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

DEV = "cuda:0"
HEADS, KV_HEADS, DIM, LAYERS, VOCAB, THETA = 16, 2, 128, 36, 151936, 1.0e6
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
CODES = {"fp32": 0, "bf16": 1, "fp16": 2}


# ------------------------------------------------------------------ cases
def listed() -> list[dict]:
    return [
        # one decode round of a small batch: the smallest call, once a layer and token
        _rope("rope 8 tokens", "bf16", 8, page=16),
        # a prompt of no round length, a model that rotates half of each head in pairs, stretched fourfold
        _rope("rope 1999 fp16 pairs", "fp16", 1999, rotary=DIM // 2, pairs=True, stretch=4.0, factor=1.1386, page=16),
        # a round of long prompt chunks of many sequences
        _rope("rope 32768 tokens", "bf16", 32768, page=64),
        # a single chat turn: one token over a middling cache, latency bound
        _attention("decode 1 x 2000", "bf16", 1, 1, 2000, page=16),
        # a decode round of a busy server, lengths as they come
        _attention("decode 64 x 8192 ragged", "bf16", 64, 1, 8191, ragged=True, page=16),
        # one token over a very long document
        _attention("decode 1 x 120000", "fp16", 1, 1, 120000, page=64),
        # a round that mixes prompt chunks with sequences that decode; small heads
        _attention("mixed 6 chunks fp16", "fp16", 6, 1500, 3000, heads=12, kv_heads=4, dim=64, ragged=True, page=16),
        # a long prompt in one piece: the largest product
        _attention("prompt 8192", "bf16", 1, 8192, 0, page=64),
        # the last pages of a round of forked sequences, all layers
        {"name": "copy 8 pages", "kind": "pages", "layers": LAYERS, "pages": 64, "moves": 8, "page": 16, "kv_heads": KV_HEADS,
         "dim": DIM},
        # compaction of a cache that many sequences have left
        {"name": "compact 200 pages", "kind": "pages", "layers": LAYERS, "pages": 500, "moves": 200, "page": 16,
         "kv_heads": KV_HEADS, "dim": DIM},
        # the next token of one sequence, the usual settings
        {"name": "sample 1 row", "kind": "sample", "dtype": "bf16", "rows": 1, "vocab": VOCAB, "mix": "top-k and top-p"},
        # a round of a busy server, every row with settings of its own
        {"name": "sample 128 rows mixed", "kind": "sample", "dtype": "bf16", "rows": 128, "vocab": VOCAB, "mix": "mixed"},
    ]


def _rope(name, dtype, tokens, heads=HEADS, kv_heads=KV_HEADS, dim=DIM, rotary=DIM, pairs=False, stretch=1.0,
          factor=1.0, page=16) -> dict:
    return {"name": name, "kind": "rope", "dtype": dtype, "tokens": tokens, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "rotary": rotary, "pairs": pairs, "stretch": stretch, "factor": factor, "page": page}


def _attention(name, dtype, sequences, new, cached, heads=HEADS, kv_heads=KV_HEADS, dim=DIM, ragged=False,
               page=16) -> dict:
    return {"name": name, "kind": "attention", "dtype": dtype, "sequences": sequences, "new": new, "cached": cached,
            "heads": heads, "kv_heads": kv_heads, "dim": dim, "ragged": ragged, "page": page}


def _spread(rng, low: int, high: int) -> int:
    """A whole number from low to high, even over its logarithm."""

    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng) -> dict:
    kind = rng.choice(["rope", "attention", "attention", "attention", "pages", "sample", "sample"])
    heads, kv_heads = rng.choice([(16, 2), (16, 2), (12, 4), (8, 8), (7, 1), (32, 8)])
    dim = rng.choice([64, 128, 128])
    page = rng.choice([1, 16, 16, 64, 256])
    if kind == "rope":
        case = _rope("", rng.choice(["bf16", "fp16"]), _spread(rng, 1, 16000), heads, kv_heads, dim,
                     rng.choice([dim, dim, dim // 2, dim // 4]), rng.random() < 0.4, rng.choice([1.0, 1.0, 4.0, 32.0]),
                     rng.choice([1.0, 1.0, 1.1386]), page)
    elif kind == "attention":
        decode = rng.random() < 0.5
        sequences = _spread(rng, 1, 64 if decode else 12)
        new = 1 if decode else _spread(rng, 1, 4000)
        # the whole cache within a busy server's, the padded products within a quarter of the longest prompt's
        room = min(60000, 75_000_000 // (sequences * kv_heads * dim), 270_000_000 // (sequences * new * heads))
        cached = 0 if room < 1 else _spread(rng, 1, room) - (rng.random() < 0.2)
        while sequences > 1 and sequences * new * heads * (new + cached) > 270_000_000:
            sequences -= 1
        case = _attention("", rng.choice(["bf16", "bf16", "fp16"]), sequences, new, cached, heads, kv_heads, dim,
                          rng.random() < 0.7, page)
    elif kind == "pages":
        pages = _spread(rng, 8, 400)
        case = {"kind": kind, "layers": rng.randint(1, LAYERS), "pages": pages, "moves": rng.randint(1, pages // 2),
                "page": rng.choice([1, 8, 16]), "kv_heads": kv_heads if kv_heads < 8 else 2, "dim": dim}
    else:
        case = {"kind": kind, "dtype": rng.choice(["bf16", "fp16", "fp32"]), "rows": _spread(rng, 1, 60),
                "vocab": _spread(rng, 1000, VOCAB),
                "mix": rng.choice(["top-k", "top-p", "top-k and top-p", "min-p", "temperature", "mixed"])}
    case.pop("name", None)
    return case


def _lengths(case) -> tuple[list[int], list[int]]:
    """New tokens and cached tokens of every sequence: the case's, or up to them, the first sequence's in full."""

    n, new, cached = case["sequences"], case["new"], case["cached"]
    if not case["ragged"]:
        return [new] * n, [cached] * n
    rng = random.Random("%d %d %d" % (n, new, cached))
    return ([new] + [_spread(rng, 1, new) for _ in range(n - 1)],
            [cached] + [rng.randint(0, cached) for _ in range(n - 1)])


def work(case) -> dict:
    """What a pass has to read, write and compute."""

    if case["kind"] == "rope":
        size, pairs = 2, case["rotary"] // 2
        row = (case["heads"] + 2 * case["kv_heads"]) * case["dim"] * size
        rotated = (case["heads"] + case["kv_heads"]) * pairs
        return {"bytes": case["tokens"] * (2 * row + 12), "flops": case["tokens"] * rotated * 6}
    if case["kind"] == "attention":
        new, cached = _lengths(case)
        row = case["kv_heads"] * case["dim"] * 2
        seen = sum(n * c + n * (n + 1) // 2 for n, c in zip(new, cached))
        rows = sum(n + c for n, c in zip(new, cached))
        return {"bytes": 2 * rows * row + 4 * sum(new) * case["heads"] * case["dim"],
                "flops": 4 * seen * case["heads"] * case["dim"]}
    if case["kind"] == "pages":
        return {"bytes": 2 * 2 * case["layers"] * case["moves"] * case["page"] * case["kv_heads"] * case["dim"] * 2,
                "flops": 0}
    return {"bytes": case["rows"] * case["vocab"] * (4 if case["dtype"] == "fp32" else 2), "flops": case["rows"] * case["vocab"]}


# ----------------------------------------------------------------- inputs
def _gen(seed: int) -> torch.Generator:
    return torch.Generator(device=DEV).manual_seed(int(seed) * 1000003 + 17)


def _normal(gen, shape, dtype, std=1.0) -> torch.Tensor:
    return (torch.randn(shape, generator=gen, device=DEV) * std).to(dtype)


def prepare(case, seed) -> dict:
    """What the program holds before the call: its pools, tables and settings, and the new inputs."""

    gen = _gen(seed)
    rng = np.random.default_rng([int(seed), 5])
    state = {"case": case}
    if case["kind"] == "rope":
        return state | _rope_inputs(case, gen, rng)
    if case["kind"] == "attention":
        return state | _attention_inputs(case, gen, rng)
    if case["kind"] == "pages":
        size = case["page"] * case["kv_heads"] * case["dim"]
        pool = _normal(gen, (2 * case["layers"], case["pages"], size), torch.bfloat16)
        order = rng.permutation(case["pages"]).astype(np.int32)
        pairs = np.stack([order[:case["moves"]], order[case["moves"]:2 * case["moves"]]], axis=1)
        return state | {"pool": pool, "pairs": np.ascontiguousarray(pairs)}
    return state | _sample_inputs(case, gen, rng)


def _rope_inputs(case, gen, rng) -> dict:
    dtype, t, d = TYPES[case["dtype"]], case["tokens"], case["dim"]
    h, g = case["heads"], case["kv_heads"]
    # the QKV projection's output: q, k and v of a token side by side
    qkv = _normal(gen, (t, (h + 2 * g) * d), dtype)
    freq = THETA ** (-np.arange(0, case["rotary"], 2, dtype=np.float64) / case["rotary"]) / case["stretch"]
    # up to eight sequences, each a run of consecutive positions
    cuts = np.sort(rng.integers(0, t, size=min(8, t) - 1)) if t > 1 else np.zeros(0, np.int64)
    starts = np.concatenate([[0], cuts, [t]])
    positions = np.concatenate([np.arange(b - a) + rng.integers(0, 100000) for a, b in zip(starts[:-1], starts[1:])])
    pages = -(-t // case["page"]) + 3
    order = rng.permutation(pages)
    at = np.arange(t)
    slots = order[at // case["page"]].astype(np.int64) * case["page"] + at % case["page"]
    shape = (pages, g, case["page"], d)
    return {"qkv": qkv, "freq": torch.from_numpy(freq).to(DEV),
            "positions": torch.from_numpy(positions.astype(np.int32)).to(DEV), "slots": torch.from_numpy(slots).to(DEV),
            "query": torch.empty((t, h, d), dtype=dtype, device=DEV),
            "keys": torch.zeros(shape, dtype=dtype, device=DEV), "values": torch.zeros(shape, dtype=dtype, device=DEV)}


def _attention_inputs(case, gen, rng) -> dict:
    dtype, d, g, page = TYPES[case["dtype"]], case["dim"], case["kv_heads"], case["page"]
    new, cached = _lengths(case)
    kv = np.array(new) + np.array(cached)
    used = -(-kv // page)
    pages = int(used.sum()) + 5
    order = rng.permutation(pages)
    table = np.zeros((case["sequences"], int(used.max())), dtype=np.int32)
    ends = np.cumsum(used)
    for i, n in enumerate(used):
        table[i, :n] = order[ends[i] - n:ends[i]]
    starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    tokens = int(starts[-1])
    # keys with channels of unlike size and a common part, as after a projection with a bias
    spread = torch.exp(torch.randn((g, 1, d), generator=gen, device=DEV) * 0.4)
    shift = torch.randn((g, 1, d), generator=gen, device=DEV) * 0.5
    keys = torch.empty((pages, g, page, d), dtype=dtype, device=DEV)
    values = torch.empty((pages, g, page, d), dtype=dtype, device=DEV)
    keys.copy_(torch.randn((pages, g, page, d), generator=gen, device=DEV) * spread + shift)
    values.copy_(torch.randn((pages, g, page, d), generator=gen, device=DEV))
    return {"query": _normal(gen, (tokens, case["heads"], d), dtype, 1.5), "keys": keys, "values": values,
            "table": torch.from_numpy(table).to(DEV), "starts": torch.from_numpy(starts).to(DEV),
            "kv_lens": torch.from_numpy(kv.astype(np.int32)).to(DEV),
            "out": torch.empty((tokens, case["heads"], d), dtype=dtype, device=DEV), "tokens": tokens,
            "max_new": max(new), "max_kv": int(kv.max()), "scale": 1.0 / math.sqrt(d)}


def _sample_inputs(case, gen, rng) -> dict:
    rows, vocab, mix = case["rows"], case["vocab"], case["mix"]
    # a broad bulk and some tokens that stand out, as logits have them
    logits = torch.randn((rows, vocab), generator=gen, device=DEV) * 2.2
    rare = torch.rand((rows, vocab), generator=gen, device=DEV)
    logits = logits + torch.where(rare < 40.0 / vocab, rare * (vocab / 40.0) * 10.0, 0.0)
    logits = logits.to(TYPES[case["dtype"]])
    temperature = np.full(rows, 0.8, np.float32)
    top_k, top_p, min_p = np.zeros(rows, np.int32), np.ones(rows, np.float32), np.zeros(rows, np.float32)
    if mix in ("top-k", "top-k and top-p"):
        top_k[:] = 50
    if mix in ("top-p", "top-k and top-p"):
        top_p[:] = 0.95
    if mix == "min-p":
        min_p[:] = 0.05
    if mix == "mixed":
        temperature = rng.choice([0.0, 0.6, 0.8, 1.0, 1.3], size=rows).astype(np.float32)
        top_k = rng.choice([0, 0, 20, 50, 400], size=rows).astype(np.int32)
        top_p = rng.choice([1.0, 0.8, 0.95, 0.99], size=rows).astype(np.float32)
        min_p = rng.choice([0.0, 0.0, 0.02, 0.1], size=rows).astype(np.float32)
    return {"logits": logits, "random": torch.rand(rows, generator=gen, device=DEV),
            "temperature": torch.from_numpy(temperature).to(DEV), "top_k": torch.from_numpy(top_k).to(DEV),
            "top_p": torch.from_numpy(top_p).to(DEV), "min_p": torch.from_numpy(min_p).to(DEV),
            "tokens": torch.empty(rows, dtype=torch.int32, device=DEV),
            "chances": torch.empty(rows, dtype=torch.float32, device=DEV)}


# ------------------------------------------------------------ plain forms
def _rotate(x, cos, sin, rotary: int, pairs: bool) -> torch.Tensor:
    """x [tokens, heads, dim] in 32 bits, cos and sin [tokens, rotary / 2]."""

    cos, sin = cos[:, None, :], sin[:, None, :]
    turned, rest = x[..., :rotary], x[..., rotary:]
    if pairs:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack([a * cos - b * sin, a * sin + b * cos], dim=-1).flatten(-2)
    else:
        a, b = turned[..., :rotary // 2], turned[..., rotary // 2:]
        turned = torch.cat([a * cos - b * sin, a * sin + b * cos], dim=-1)
    return torch.cat([turned, rest], dim=-1)


def _plain_rope(s) -> dict:
    case = s["case"]
    h, g, d, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    angle = s["positions"].double()[:, None] * s["freq"][None, :]
    cos, sin = (angle.cos() * case["factor"]).float(), (angle.sin() * case["factor"]).float()
    q, k, v = s["qkv"].float().view(-1, h + 2 * g, d).split([h, g, g], dim=1)
    query = _rotate(q, cos, sin, case["rotary"], case["pairs"]).to(s["qkv"].dtype)
    k = _rotate(k, cos, sin, case["rotary"], case["pairs"]).to(s["qkv"].dtype)
    at, offset = s["slots"] // page, s["slots"] % page
    s["keys"][at, :, offset] = k
    s["values"][at, :, offset] = v.to(s["qkv"].dtype)
    return {"query": query, "keys": s["keys"], "values": s["values"]}


def _plain_attention(s) -> dict:
    """All sequences at once, padded to the longest."""

    case = s["case"]
    h, g, d, n = case["heads"], case["kv_heads"], case["dim"], case["sequences"]
    table, starts, kv_lens = s["table"].long(), s["starts"].long(), s["kv_lens"].long()
    rows = table.shape[1] * case["page"]
    k = s["keys"][table].float().transpose(1, 2).reshape(n, g, rows, d)
    v = s["values"][table].float().transpose(1, 2).reshape(n, g, rows, d)
    new = starts[1:] - starts[:-1]
    at = torch.arange(s["max_new"], device=DEV)
    token = torch.minimum(starts[:-1, None] + at, starts[1:, None] - 1)
    q = s["query"].float()[token]  # [n, max_new, h, d]
    q = q.view(n, s["max_new"], g, h // g, d).permute(0, 2, 3, 1, 4).reshape(n, g, h // g * s["max_new"], d)
    scores = torch.matmul(q, k.transpose(2, 3).contiguous()) * s["scale"]
    scores = scores.view(n, g, h // g, s["max_new"], rows)
    last = (kv_lens - new)[:, None] + at  # the position that a row may look up to
    hidden = torch.arange(rows, device=DEV) > last[:, :, None]
    scores = scores.masked_fill(hidden[:, None, None], -math.inf)
    top = scores.amax(dim=-1, keepdim=True)
    scores = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = scores.sum(dim=-1, keepdim=True)
    out = torch.matmul(scores.view(n, g, h // g * s["max_new"], rows), v).view(n, g, h // g, s["max_new"], d)
    out = torch.where(total == 0, 0.0, out / total).permute(0, 3, 1, 2, 4).reshape(n, s["max_new"], h, d)
    order = torch.arange(s["tokens"], device=DEV)
    of = torch.searchsorted(starts[1:], order, right=True)
    return {"out": out[of, order - starts[of]].to(s["query"].dtype)}


def _plain_pages(s) -> dict:
    pairs = torch.from_numpy(s["pairs"]).to(DEV).long()
    s["pool"][:, pairs[:, 1]] = s["pool"][:, pairs[:, 0]]
    return {"pool": s["pool"]}


def _plain_sample(s) -> dict:
    x = s["logits"].double()
    greedy = s["temperature"] <= 0
    x = x / torch.where(greedy, 1.0, s["temperature"]).double()[:, None]
    vocab = x.shape[1]
    ordered, index = torch.sort(x, dim=1, descending=True, stable=True)
    weight = torch.exp(ordered - ordered[:, :1])
    rank = torch.arange(vocab, device=DEV)
    top_k = torch.where(s["top_k"] <= 0, vocab, s["top_k"])
    weight = torch.where(rank < top_k[:, None], weight, 0.0)
    total = weight.cumsum(dim=1)
    before = total - weight
    top_p = s["top_p"].double()[:, None]
    keep = (weight > 0) & ((before < top_p * total[:, -1:]) | (top_p >= 1)) & (weight >= s["min_p"].double()[:, None])
    keep[:, 0] = True
    weight = torch.zeros_like(x).scatter_(1, index, torch.where(keep, weight, 0.0))
    total = weight.cumsum(dim=1)
    token = (total <= s["random"].double()[:, None] * total[:, -1:]).sum(dim=1)
    chance = weight.gather(1, token.clamp(max=vocab - 1)[:, None])[:, 0] / total[:, -1]
    return {"tokens": torch.where(greedy, index[:, 0], token).to(torch.int32),
            "chances": torch.where(greedy, 1.0, chance).float()}


# ---------------------------------------------------- the framework's calls
_program: dict = {}


def _native():
    """The program's one handle."""

    if "native" not in _program:
        from kudacuda_amd._native import Native

        _program["native"] = Native(0)
    return _program["native"]


def _workspace(nbytes: int) -> torch.Tensor:
    """The program's one workspace, as large as its calls have needed so far."""

    if "workspace" not in _program or _program["workspace"].numel() < nbytes:
        _program["workspace"] = torch.empty(nbytes, dtype=torch.uint8, device=DEV)
    return _program["workspace"]


def _own_rope(s) -> dict:
    case, qkv, keys = s["case"], s["qkv"], s["keys"]
    h, g, d = case["heads"], case["kv_heads"], case["dim"]
    base = qkv.data_ptr()
    row = qkv.stride(0)
    _native().call("kudacuda_rope_paged_append", base, base + 2 * h * d, base + 2 * (h + g) * d, s["freq"].data_ptr(),
                   s["positions"].data_ptr(), s["slots"].data_ptr(), s["query"].data_ptr(), keys.data_ptr(),
                   s["values"].data_ptr(), CODES[case["dtype"]], case["tokens"], h, g, d, case["rotary"],
                   int(case["pairs"]), row, row, row, h * d, keys.shape[0], case["page"], keys.stride(0),
                   keys.stride(1), keys.stride(2), case["factor"], torch.cuda.current_stream().cuda_stream)
    return {"query": s["query"], "keys": keys, "values": s["values"]}


def _own_attention(s) -> dict:
    case, keys, native = s["case"], s["keys"], _native()
    h, g, d, n = case["heads"], case["kv_heads"], case["dim"], case["sequences"]
    nbytes = native.lib.kudacuda_paged_attention_workspace_bytes(s["tokens"], n, s["max_new"], s["max_kv"], h, g, d)
    native.call("kudacuda_paged_attention", s["query"].data_ptr(), keys.data_ptr(), s["values"].data_ptr(),
                s["table"].data_ptr(), s["starts"].data_ptr(), s["kv_lens"].data_ptr(), s["out"].data_ptr(),
                _workspace(nbytes).data_ptr(), nbytes, CODES[case["dtype"]], s["tokens"], n, s["max_new"], s["max_kv"],
                h, g, d, h * d, h * d, keys.shape[0], case["page"], s["table"].shape[1], keys.stride(0),
                keys.stride(1), keys.stride(2), s["scale"], torch.cuda.current_stream().cuda_stream)
    return {"out": s["out"]}


def _own_pages(s) -> dict:
    pool, pairs = s["pool"], s["pairs"]
    _native().call("kudacuda_copy_pages", pool.data_ptr(), pairs.ctypes.data, len(pairs), pool.shape[0], pool.shape[1],
                   2 * pool.shape[2], 2 * pool.stride(1), 2 * pool.stride(0), torch.cuda.current_stream().cuda_stream)
    return {"pool": pool}


def _own_sample(s) -> dict:
    logits, native = s["logits"], _native()
    rows, vocab = logits.shape
    nbytes = native.lib.kudacuda_sample_workspace_bytes(rows, vocab)
    native.call("kudacuda_sample_tokens", logits.data_ptr(), s["random"].data_ptr(), s["temperature"].data_ptr(),
                s["top_k"].data_ptr(), s["top_p"].data_ptr(), s["min_p"].data_ptr(), s["tokens"].data_ptr(),
                s["chances"].data_ptr(), _workspace(nbytes).data_ptr(), nbytes, CODES[s["case"]["dtype"]], rows, vocab,
                logits.stride(0), torch.cuda.current_stream().cuda_stream)
    return {"tokens": s["tokens"], "chances": s["chances"]}


def run(state) -> dict:
    kind = state["case"]["kind"]
    if own:
        return {"rope": _own_rope, "attention": _own_attention, "pages": _own_pages, "sample": _own_sample}[kind](state)
    return {"rope": _plain_rope, "attention": _plain_attention, "pages": _plain_pages, "sample": _plain_sample}[kind](state)


# ----------------------------------------------------------------- 64 bits
def exact(case, seed):
    """Rotated rows, attention and chances in 64 bits; copied rows, pages and token ids are not computed numbers."""

    if case["kind"] == "rope":
        return _exact_rope(prepare(case, seed))
    if case["kind"] == "attention":
        return _exact_attention(prepare(case, seed))
    return _exact_sample(prepare(case, seed)) if case["kind"] == "sample" else None


def _exact_rope(s) -> dict:
    """Each pair as a complex number times its turn."""

    case = s["case"]
    h, g, d, r = case["heads"], case["kv_heads"], case["dim"], case["rotary"]
    turn = torch.polar(torch.full((), case["factor"], dtype=torch.float64, device=DEV),
                       torch.outer(s["positions"].double(), s["freq"]))
    qkv = s["qkv"].double().view(-1, h + 2 * g, d)
    first = torch.arange(r // 2, device=DEV) * (2 if case["pairs"] else 1)
    second = first + (1 if case["pairs"] else r // 2)
    product = torch.complex(qkv[:, :h + g, first], qkv[:, :h + g, second]) * turn[:, None]
    rows = qkv[:, :h + g].clone()
    rows[:, :, first], rows[:, :, second] = product.real.clone(), product.imag.clone()
    keys = torch.zeros(s["keys"].shape, dtype=torch.float64, device=DEV)
    by_row = keys.transpose(1, 2).reshape(-1, g, d)
    by_row[s["slots"]] = rows[:, h:]
    keys = by_row.view(keys.shape[0], case["page"], g, d).transpose(1, 2)
    return {"query": rows[:, :h].contiguous(), "keys": keys.contiguous(), "values": None}


def _exact_attention(s) -> dict:
    """Sequence by sequence and head by head."""

    case = s["case"]
    h, g, page = case["heads"], case["kv_heads"], case["page"]
    new, cached = _lengths(case)
    out = torch.empty(s["query"].shape, dtype=torch.float64, device=DEV)
    begin = 0
    for i, (n, c) in enumerate(zip(new, cached)):
        pages = s["table"][i, :-(-(n + c) // page)].long()
        see = torch.ones((n, n + c), dtype=torch.bool, device=DEV).tril(c)
        for head in range(h):
            k = s["keys"][pages, head // (h // g)].double().flatten(0, 1)[:n + c]
            v = s["values"][pages, head // (h // g)].double().flatten(0, 1)[:n + c]
            scores = (s["query"][begin:begin + n, head].double() @ k.T) * s["scale"]
            out[begin:begin + n, head] = torch.softmax(scores.masked_fill(~see, -math.inf), dim=1) @ v
        begin += n
    return {"out": out}


def _exact_sample(s) -> dict:
    """Row by row, token by token down the order."""

    logits = s["logits"].double().cpu().numpy()
    settings = [s[n].double().cpu().numpy() for n in ("temperature", "top_k", "top_p", "min_p", "random")]
    chances = np.ones(len(logits))
    for i, (heat, top_k, top_p, min_p, u) in enumerate(zip(*settings)):
        if heat <= 0:
            continue
        order = np.argsort(-logits[i], kind="stable")
        order = order[:int(top_k)] if top_k > 0 else order
        p = np.exp((logits[i][order] - logits[i][order[0]]) / heat)
        kept = np.count_nonzero(np.cumsum(p) - p < top_p * p.sum()) if top_p < 1 else len(p)
        kept = max(1, min(kept, np.count_nonzero(p >= min_p)))
        ids, p = order[:kept], p[:kept] / p[:kept].sum()
        by_id = np.argsort(ids)
        chances[i] = p[by_id][np.searchsorted(np.cumsum(p[by_id]), u, side="right")]
    return {"tokens": None, "chances": torch.from_numpy(chances)}
