"""A paged KV cache held in 4 or 8 bits, and the adapters of many requests, as cases that can be timed and compared.

A server whose caches fill the card keeps them in microscaled numbers: blocks of 32
dims of a row share a power of two (one byte, 127 + exponent; 0 for a block of zeros,
255 for NaN), their elements are e2m1 (4 bits, the even dim in the low half of a byte)
or e4m3 (8 bits).
A page holds the elements [kv_heads, page_size, dim] and behind them the blocks' bytes
[kv_heads, page_size, dim / 32].

* ``append`` -- rotate new queries and keys, write keys and values into their pages
  (``kudacuda_rope_paged_append_mx``), and read back what the cache now holds for them
  (``kudacuda_paged_read_mx``);
* ``read`` -- read rows back from their pages, to move a sequence elsewhere
  (``kudacuda_paged_read_mx``);
* ``attention`` -- attend from the new tokens of every sequence to all of its pages
  (``kudacuda_paged_attention_mx``);
* ``adapters`` -- add to a shared projection's rows what each request's own low-rank
  adapter makes of the projection's input (``kudacuda_lora_add``).

With ``own`` false, ``run`` computes them in elementary torch operations, in 32 bits
(the rotation of keys, whose rounding decides between neighbouring codes, in 64).
"""

from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

DEV = "cuda:0"
HEADS, KV_HEADS, DIM, HIDDEN, INTERMEDIATE, THETA = 16, 2, 128, 2048, 11008, 1.0e6
BLOCK = 32  # dims that share a power of two
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
CODES = {"bf16": 1, "fp16": 2}
# the lowest power of two that a block of 4 or 8 bits has: its elements are numbers of the type
LOWEST = {("bf16", 4): -110, ("bf16", 8): -110, ("fp16", 4): -23, ("fp16", 8): -15}
TILE = 64  # rows of an adapter's tile
FACTOR = float(np.float32(1.1386))  # an amplitude that scaled frequencies bring, as calls take it: in 32 bits


# ------------------------------------------------------------------ cases
def listed() -> list[dict]:
    return [
        # one decode round of a small batch: the smallest call, once a layer and token
        _append("append 8 tokens", "bf16", 4, 8),
        # a round of prompt chunks, a model that rotates half of each head in pairs, stretched fourfold
        _append("append 19999 fp16 pairs 8 bits", "fp16", 8, 19999, rotary=DIM // 2, pairs=True, stretch=4.0, factor=FACTOR),
        # a short sequence that moves to another cache
        _read("read 2000 tokens", "bf16", 4, 2000),
        # a long one
        _read("read 120000 tokens 8 bits", "bf16", 8, 120000, page=64),
        # a single chat turn: one token over a middling cache, latency bound
        _attention("decode 1 x 2000", "bf16", 4, 1, 1, 2000),
        # a decode round of a busy server, lengths as they come
        _attention("decode 64 x 8192 ragged", "bf16", 4, 64, 1, 8191, ragged=True),
        # one token over a very long document
        _attention("decode 1 x 120000 fp16 8 bits", "fp16", 8, 1, 1, 120000, page=64),
        # a round that mixes prompt chunks with sequences that decode; small heads
        _attention("mixed 6 chunks fp16", "fp16", 4, 6, 1500, 3000, heads=12, kv_heads=4, dim=64, ragged=True),
        # a long prompt in one piece: the largest product
        _attention("prompt 8192 8 bits", "bf16", 8, 1, 8192, 0, page=64),
        # the next token of one request with an adapter, beside its query projection
        _adapters("adapter 1 token", "bf16", [1], 1, HIDDEN, HIDDEN, [16]),
        # a decode round of 64 requests, each with its own adapter, beside the gate projection
        _adapters("64 adapters 64 tokens", "bf16", [1] * 64, 64, HIDDEN, INTERMEDIATE, [8, 16, 32, 64]),
        # prompt chunks of eight requests, two of them without an adapter, beside the down projection
        _adapters("8 chunks fp16", "fp16", [701, 64, 33, 1000, 1, 517, 250, 430], 6, INTERMEDIATE, HIDDEN, [16, 32]),
    ]


def _append(name, dtype, bits, tokens, heads=HEADS, kv_heads=KV_HEADS, dim=DIM, rotary=DIM, pairs=False, stretch=1.0,
            factor=1.0, page=16) -> dict:
    return {"name": name, "kind": "append", "dtype": dtype, "bits": bits, "tokens": tokens, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "rotary": rotary, "pairs": pairs, "stretch": stretch, "factor": factor,
            "page": page}


def _read(name, dtype, bits, tokens, kv_heads=KV_HEADS, dim=DIM, page=16) -> dict:
    return {"name": name, "kind": "read", "dtype": dtype, "bits": bits, "tokens": tokens, "kv_heads": kv_heads, "dim": dim,
            "page": page}


def _attention(name, dtype, bits, sequences, new, cached, heads=HEADS, kv_heads=KV_HEADS, dim=DIM, ragged=False,
               page=16) -> dict:
    return {"name": name, "kind": "attention", "dtype": dtype, "bits": bits, "sequences": sequences, "new": new,
            "cached": cached, "heads": heads, "kv_heads": kv_heads, "dim": dim, "ragged": ragged, "page": page}


def _adapters(name, dtype, chunks, adapters, inner, outer, ranks) -> dict:
    """Chunks of tokens of one request each; requests take the adapters in turn, those past them none."""

    return {"name": name, "kind": "adapters", "dtype": dtype, "chunks": ",".join(map(str, chunks)), "adapters": adapters,
            "in": inner, "out": outer, "ranks": ",".join(map(str, ranks))}


def _spread(rng, low: int, high: int) -> int:
    """A whole number from low to high, even over its logarithm."""

    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng) -> dict:
    kind = rng.choice(["append", "read", "attention", "attention", "attention", "adapters", "adapters"])
    heads, kv_heads = rng.choice([(16, 2), (16, 2), (12, 4), (8, 8), (7, 1), (32, 8)])
    dim = rng.choice([64, 128, 128])
    page = rng.choice([16, 16, 64, 256])
    bits = rng.choice([4, 4, 8])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if kind == "append":
        case = _append("", dtype, bits, _spread(rng, 1, 16000), heads, kv_heads, dim,
                       rng.choice([dim, dim, dim // 2, dim // 4]), rng.random() < 0.4, rng.choice([1.0, 1.0, 4.0, 32.0]),
                       rng.choice([1.0, 1.0, FACTOR]), page)
    elif kind == "read":
        case = _read("", dtype, bits, _spread(rng, 1, 60000 // kv_heads), kv_heads, dim, page)
    elif kind == "attention":
        decode = rng.random() < 0.5
        sequences = _spread(rng, 1, 64 if decode else 12)
        new = 1 if decode else _spread(rng, 1, 4000)
        # the whole cache within a busy server's, the padded products within a quarter of the longest prompt's
        room = min(60000, 75_000_000 // (sequences * kv_heads * dim), 270_000_000 // (sequences * new * heads))
        cached = 0 if room < 1 else _spread(rng, 1, room) - (rng.random() < 0.2)
        while sequences > 1 and sequences * new * heads * (new + cached) > 270_000_000:
            sequences -= 1
        case = _attention("", dtype, bits, sequences, new, cached, heads, kv_heads, dim, rng.random() < 0.7, page)
    else:
        requests = _spread(rng, 1, 64)
        longest = 1 if rng.random() < 0.5 else _spread(rng, 1, max(1, 3000 // requests))
        chunks = [_spread(rng, 1, longest) for _ in range(requests)]
        ranks = rng.choice([[16], [8], [64], [8, 16, 32, 64], [4, 12, 24], [128], [1, 40]])
        case = _adapters("", dtype, chunks, _spread(rng, 1, requests), 8 * _spread(rng, 8, INTERMEDIATE // 8),
                         8 * _spread(rng, 8, INTERMEDIATE // 8), ranks)
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


def _numbers(text: str) -> list[int]:
    return [int(x) for x in text.split(",")]


def _ranks(case) -> list[int]:
    """The rank of every adapter: the case's in turn."""

    ranks = _numbers(case["ranks"])
    return [ranks[i % len(ranks)] for i in range(case["adapters"])]


def _row_bytes(case) -> int:
    """A head's row in the cache: its elements and its blocks' powers of two."""

    return case["dim"] * case["bits"] // 8 + case["dim"] // BLOCK


def work(case) -> dict:
    """What a pass has to read, write and compute."""

    if case["kind"] == "append":
        h, g, d, pairs = case["heads"], case["kv_heads"], case["dim"], case["rotary"] // 2
        # projections read; queries, cache and the cache's rows written
        row = 2 * (h + 2 * g) * d + 2 * h * d + 2 * g * _row_bytes(case) + 2 * 2 * g * d
        return {"bytes": case["tokens"] * (row + 12), "flops": case["tokens"] * (h + g) * pairs * 6}
    if case["kind"] == "read":
        row = 2 * case["kv_heads"] * (_row_bytes(case) + 2 * case["dim"])
        return {"bytes": case["tokens"] * (row + 8), "flops": case["tokens"] * 2 * case["kv_heads"] * case["dim"]}
    if case["kind"] == "attention":
        new, cached = _lengths(case)
        seen = sum(n * c + n * (n + 1) // 2 for n, c in zip(new, cached))
        rows = sum(n + c for n, c in zip(new, cached))
        return {"bytes": 2 * rows * case["kv_heads"] * _row_bytes(case) + 4 * sum(new) * case["heads"] * case["dim"],
                "flops": 4 * seen * case["heads"] * case["dim"]}
    chunks, ranks = _numbers(case["chunks"]), _ranks(case)
    tokens, inner, outer = sum(chunks), case["in"], case["out"]
    served = [n for i, n in enumerate(chunks) if i < case["adapters"]]
    return {"bytes": 2 * (sum(served) * inner + 2 * tokens * outer + sum(ranks[:len(served)]) * (inner + outer)),
            "flops": sum(2 * n * r * (inner + outer) for n, r in zip(served, ranks))}


# ----------------------------------------------------------------- inputs
def _gen(seed: int) -> torch.Generator:
    return torch.Generator(device=DEV).manual_seed(int(seed) * 1000003 + 29)


def _normal(gen, shape, dtype, std=1.0) -> torch.Tensor:
    return (torch.randn(shape, generator=gen, device=DEV) * std).to(dtype)


def _pools(case, pages: int) -> tuple[torch.Tensor, torch.Tensor]:
    """Empty pools of bytes, [pages, bytes of a page]."""

    shape = (pages, case["kv_heads"] * case["page"] * _row_bytes(case))
    return torch.zeros(shape, dtype=torch.uint8, device=DEV), torch.zeros(shape, dtype=torch.uint8, device=DEV)


def _parts(case, pool) -> tuple[torch.Tensor, torch.Tensor]:
    """A pool's elements [pages, kv_heads, page, bytes of a row] and blocks' bytes [pages, kv_heads, page, blocks]."""

    g, page = case["kv_heads"], case["page"]
    row = case["dim"] * case["bits"] // 8
    elements = pool[:, :g * page * row].unflatten(1, (g, page, row))
    return elements, pool[:, g * page * row:].unflatten(1, (g, page, case["dim"] // BLOCK))


def prepare(case, seed) -> dict:
    """What the program holds before the call: its pools, tables, adapters and plans, and the new inputs."""

    gen = _gen(seed)
    rng = np.random.default_rng([int(seed), 7])
    make = {"append": _append_inputs, "read": _read_inputs, "attention": _attention_inputs, "adapters": _adapter_inputs}
    return {"case": case} | make[case["kind"]](case, gen, rng)


def _slots(case, rng) -> tuple[torch.Tensor, int]:
    """Places of the case's tokens in pages in no order, and how many pages there are."""

    t, page = case["tokens"], case["page"]
    pages = -(-t // page) + 3
    order = rng.permutation(pages)
    at = np.arange(t)
    return torch.from_numpy(order[at // page].astype(np.int64) * page + at % page).to(DEV), pages


def _append_inputs(case, gen, rng) -> dict:
    dtype, t, d = TYPES[case["dtype"]], case["tokens"], case["dim"]
    h, g = case["heads"], case["kv_heads"]
    # the QKV projection's output: q, k and v of a token side by side, channels of unlike size
    qkv = torch.randn((t, (h + 2 * g) * d), generator=gen, device=DEV)
    qkv = (qkv * torch.exp(torch.randn(qkv.shape[1], generator=gen, device=DEV) * 0.5)).to(dtype)
    freq = THETA ** (-np.arange(0, case["rotary"], 2, dtype=np.float64) / case["rotary"]) / case["stretch"]
    # up to eight sequences, each a run of consecutive positions
    cuts = np.sort(rng.integers(0, t, size=min(8, t) - 1)) if t > 1 else np.zeros(0, np.int64)
    starts = np.concatenate([[0], cuts, [t]])
    positions = np.concatenate([np.arange(b - a) + rng.integers(0, 100000) for a, b in zip(starts[:-1], starts[1:])])
    slots, pages = _slots(case, rng)
    keys, values = _pools(case, pages)
    return {"qkv": qkv, "freq": torch.from_numpy(freq).to(DEV),
            "positions": torch.from_numpy(positions.astype(np.int32)).to(DEV), "slots": slots,
            "query": torch.empty((t, h, d), dtype=dtype, device=DEV), "keys": keys, "values": values,
            "key_rows": torch.empty((t, g, d), dtype=dtype, device=DEV),
            "value_rows": torch.empty((t, g, d), dtype=dtype, device=DEV)}


def _fill(case, pool, gen, spread: float, shift: float) -> None:
    """Random rows of unlike channels and a common part, as after a projection with a bias, in the pool's numbers."""

    elements, blocks = _parts(case, pool)
    pages, g, page, _ = elements.shape
    scale = torch.exp(torch.randn((g, 1, case["dim"]), generator=gen, device=DEV) * spread)
    common = torch.randn((g, 1, case["dim"]), generator=gen, device=DEV) * shift
    step = max(1, 40_000_000 // (g * page * case["dim"]))
    for i in range(0, pages, step):
        n = min(step, pages - i)
        x = torch.randn((n, g, page, case["dim"]), generator=gen, device=DEV) * scale + common
        packed, powers = _to_cache(x.to(TYPES[case["dtype"]]).float(), case)
        elements[i:i + n], blocks[i:i + n] = packed, powers


def _read_inputs(case, gen, rng) -> dict:
    slots, pages = _slots(case, rng)
    keys, values = _pools(case, pages)
    _fill(case, keys, gen, 0.4, 0.5)
    _fill(case, values, gen, 0.0, 0.0)
    rows = (case["tokens"], case["kv_heads"], case["dim"])
    return {"slots": slots, "keys": keys, "values": values,
            "key_rows": torch.empty(rows, dtype=TYPES[case["dtype"]], device=DEV),
            "value_rows": torch.empty(rows, dtype=TYPES[case["dtype"]], device=DEV)}


def _attention_inputs(case, gen, rng) -> dict:
    dtype, d, page = TYPES[case["dtype"]], case["dim"], case["page"]
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
    keys, values = _pools(case, pages)
    _fill(case, keys, gen, 0.4, 0.5)
    _fill(case, values, gen, 0.0, 0.0)
    return {"query": _normal(gen, (tokens, case["heads"], d), dtype, 1.5), "keys": keys, "values": values,
            "table": torch.from_numpy(table).to(DEV), "starts": torch.from_numpy(starts).to(DEV),
            "kv_lens": torch.from_numpy(kv.astype(np.int32)).to(DEV),
            "out": torch.empty((tokens, case["heads"], d), dtype=dtype, device=DEV), "tokens": tokens,
            "max_new": max(new), "max_kv": int(kv.max()), "scale": 1.0 / math.sqrt(d)}


def _adapter_inputs(case, gen, rng) -> dict:
    dtype, n, inner, outer = TYPES[case["dtype"]], case["adapters"], case["in"], case["out"]
    chunks, ranks = _numbers(case["chunks"]), _ranks(case)
    tokens, most = sum(chunks), -(-max(ranks) // 8) * 8
    # trained adapters: rows of the first factor as wide as an initial projection's, the second's small
    down = _normal(gen, (n, most, inner), dtype, inner**-0.5)
    up = _normal(gen, (n, outer, most), dtype, 0.02)
    laid = torch.zeros((n, outer * most), dtype=dtype, device=DEV)  # each adapter's rows as long as its own rank
    for i, r in enumerate(ranks):
        down[i, r:] = 0
        up[i, :, r:] = 0
        pitch = -(-r // 8) * 8
        laid[i, :outer * pitch] = up[i, :, :pitch].reshape(-1)
    # the round's plan: token rows in the order of their adapters, tiles of one adapter's rows
    of = np.repeat([i if i < n else -1 for i in range(len(chunks))], chunks)
    order = np.argsort(of, kind="stable").astype(np.int32)
    tiles = []
    for a in np.unique(of):
        first, count = np.searchsorted(of[order], a), np.count_nonzero(of == a)
        tiles += [(a, first + i, min(TILE, count - i)) for i in range(0, count, TILE)]
    tiles = np.array(tiles, dtype=np.int32)
    return {"x": _normal(gen, (tokens, inner), dtype), "base": _normal(gen, (tokens, outer), dtype),
            "down": down, "up": up, "laid": laid, "ranks": torch.tensor(ranks, dtype=torch.int32, device=DEV),
            "scales": torch.rand(n, generator=gen, device=DEV) * 2 + 0.5, "order": torch.from_numpy(order).to(DEV),
            "tiles": torch.from_numpy(tiles).to(DEV), "longest": int(tiles[:, 2].max()),
            "out": torch.empty((tokens, outer), dtype=dtype, device=DEV)}


# ------------------------------------------------------------ plain forms
def _power(exponent) -> torch.Tensor:
    """2^exponent in 32 bits, 0 for -127."""

    return ((exponent.int() + 127) << 23).view(torch.float32)


def _to_cache(x, case) -> tuple[torch.Tensor, torch.Tensor]:
    """x [..., dim] in 32 bits as the cache's bytes: elements [..., bytes of a row] and blocks' powers [..., blocks]."""

    bits = case["bits"]
    x = x.unflatten(-1, (-1, BLOCK))
    top = x.abs().amax(dim=-1)
    part, power = torch.frexp(top)  # top = part * 2^power, part in [0.5, 1)
    # the least power with top < 7 * 2^power (4 bits), 464 * 2^power (8 bits): nothing is off by more than half a step
    power = torch.where(part < 0.875, power - 3, power - 2) if bits == 4 else torch.where(part < 0.90625, power - 9, power - 8)
    power = torch.where(top == 0, -1000, power).clamp(min=LOWEST[case["dtype"], bits])
    finite = torch.isfinite(top)
    x = torch.where(finite[..., None], x * _power(-power)[..., None], 0.0)
    blocks = torch.where(finite, power + 127, 255).to(torch.uint8)
    if bits == 8:
        return x.to(torch.float8_e4m3fn).view(torch.uint8).flatten(-2), blocks
    m = x.abs()
    code = ((m > 0.25).to(torch.uint8) + (m >= 0.75).to(torch.uint8) + (m > 1.25).to(torch.uint8)
            + (m >= 1.75).to(torch.uint8) + (m > 2.5).to(torch.uint8) + (m >= 3.5).to(torch.uint8)
            + (m > 5.0).to(torch.uint8) + 8 * torch.signbit(x).to(torch.uint8)).flatten(-2)
    return code[..., 0::2] + 16 * code[..., 1::2], blocks


def _from_cache(elements, blocks, case) -> torch.Tensor:
    """What the cache's bytes stand for, [..., dim] in 32 bits."""

    if case["bits"] == 8:
        x = elements.view(torch.float8_e4m3fn).float()
    else:
        levels = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
        table = torch.tensor(levels + [-v for v in levels], device=elements.device)
        x = table[torch.stack([elements & 15, elements >> 4], dim=-1).flatten(-2).int()]
    power = torch.where(blocks == 255, math.nan, _power(blocks.int() - 127))
    return (x.unflatten(-1, (-1, BLOCK)) * power[..., None]).flatten(-2)


def _rotate(x, cos, sin, rotary: int, pairs: bool) -> torch.Tensor:
    """x [tokens, heads, dim] in the type of cos and sin, [tokens, rotary / 2]."""

    cos, sin = cos[:, None, :], sin[:, None, :]
    turned, rest = x[..., :rotary], x[..., rotary:]
    if pairs:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack([a * cos - b * sin, a * sin + b * cos], dim=-1).flatten(-2)
    else:
        a, b = turned[..., :rotary // 2], turned[..., rotary // 2:]
        turned = torch.cat([a * cos - b * sin, a * sin + b * cos], dim=-1)
    return torch.cat([turned, rest], dim=-1)


def _plain_append(s) -> dict:
    case, dtype = s["case"], s["qkv"].dtype
    h, g, d, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    angle = s["positions"].double()[:, None] * s["freq"][None, :]
    cos, sin = angle.cos() * case["factor"], angle.sin() * case["factor"]
    q, k, v = s["qkv"].view(-1, h + 2 * g, d).split([h, g, g], dim=1)
    query = _rotate(q.float(), cos.float(), sin.float(), case["rotary"], case["pairs"]).to(dtype)
    k = _rotate(k.double(), cos, sin, case["rotary"], case["pairs"]).float().to(dtype)
    at, offset = s["slots"] // page, s["slots"] % page
    for pool, x in ((s["keys"], k), (s["values"], v)):
        elements, blocks = _parts(case, pool)
        elements[at, :, offset], blocks[at, :, offset] = _to_cache(x.float(), case)
    return {"query": query} | _plain_read(s)


def _plain_read(s) -> dict:
    case, page = s["case"], s["case"]["page"]
    at, offset = s["slots"] // page, s["slots"] % page
    rows = []
    for pool in (s["keys"], s["values"]):
        elements, blocks = _parts(case, pool)
        rows.append(_from_cache(elements[at, :, offset], blocks[at, :, offset], case).to(TYPES[case["dtype"]]))
    return {"keys": rows[0], "values": rows[1]}


def _plain_attention(s) -> dict:
    """All sequences at once, padded to the longest."""

    case = s["case"]
    h, g, d, n = case["heads"], case["kv_heads"], case["dim"], case["sequences"]
    table, starts, kv_lens = s["table"].long(), s["starts"].long(), s["kv_lens"].long()
    rows = table.shape[1] * case["page"]
    k, v = (_from_cache(*(part[table] for part in _parts(case, pool)), case).transpose(1, 2).reshape(n, g, rows, d)
            for pool in (s["keys"], s["values"]))
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


def _plain_adapters(s) -> dict:
    """All tiles at once, padded to the longest; rows without an adapter meet factors of zero."""

    adapter, first, count = s["tiles"].long().unbind(dim=1)
    at = torch.arange(s["longest"], device=DEV)
    live = at < count[:, None]
    row = s["order"].long()[torch.where(live, first[:, None] + at, first[:, None])]
    some = adapter >= 0
    adapter = adapter.clamp(min=0)
    down = s["down"][adapter].float().transpose(1, 2).contiguous()
    inner = torch.matmul(s["x"][row].float(), down)
    factor = torch.where(some, s["scales"][adapter], 0.0)[:, None, None]
    delta = torch.matmul(inner, s["up"][adapter].float().transpose(1, 2).contiguous()) * factor
    out = torch.empty_like(s["base"])
    out[row[live]] = (s["base"][row[live]].float() + delta[live]).to(out.dtype)
    return {"out": out}


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


def _own_append(s) -> dict:
    case, qkv, keys = s["case"], s["qkv"], s["keys"]
    h, g, d = case["heads"], case["kv_heads"], case["dim"]
    base = qkv.data_ptr()
    row = qkv.stride(0)
    _native().call("kudacuda_rope_paged_append_mx", base, base + 2 * h * d, base + 2 * (h + g) * d, s["freq"].data_ptr(),
                   s["positions"].data_ptr(), s["slots"].data_ptr(), s["query"].data_ptr(), keys.data_ptr(),
                   s["values"].data_ptr(), CODES[case["dtype"]], case["bits"], case["tokens"], h, g, d, case["rotary"],
                   int(case["pairs"]), row, row, row, h * d, keys.shape[0], case["page"], keys.stride(0),
                   case["factor"], torch.cuda.current_stream().cuda_stream)
    return {"query": s["query"]} | _own_read(s)


def _own_read(s) -> dict:
    case, keys, rows = s["case"], s["keys"], s["key_rows"]
    _native().call("kudacuda_paged_read_mx", keys.data_ptr(), s["values"].data_ptr(), s["slots"].data_ptr(),
                   rows.data_ptr(), s["value_rows"].data_ptr(), CODES[case["dtype"]], case["bits"], case["tokens"],
                   case["kv_heads"], case["dim"], rows.stride(0), rows.stride(0), keys.shape[0], case["page"],
                   keys.stride(0), torch.cuda.current_stream().cuda_stream)
    return {"keys": rows, "values": s["value_rows"]}


def _own_attention(s) -> dict:
    case, keys, native = s["case"], s["keys"], _native()
    h, g, d, n = case["heads"], case["kv_heads"], case["dim"], case["sequences"]
    nbytes = native.lib.kudacuda_paged_attention_mx_workspace_bytes(case["bits"], s["tokens"], n, s["max_new"],
                                                                    s["max_kv"], h, g, d)
    native.call("kudacuda_paged_attention_mx", s["query"].data_ptr(), keys.data_ptr(), s["values"].data_ptr(),
                s["table"].data_ptr(), s["starts"].data_ptr(), s["kv_lens"].data_ptr(), s["out"].data_ptr(),
                _workspace(nbytes).data_ptr(), nbytes, CODES[case["dtype"]], case["bits"], s["tokens"], n, s["max_new"],
                s["max_kv"], h, g, d, h * d, h * d, keys.shape[0], case["page"], s["table"].shape[1], keys.stride(0),
                s["scale"], torch.cuda.current_stream().cuda_stream)
    return {"out": s["out"]}


def _own_adapters(s) -> dict:
    x, base, out, native = s["x"], s["base"], s["out"], _native()
    adapters, most, inner = s["down"].shape
    tiles = s["tiles"].shape[0]
    nbytes = native.lib.kudacuda_lora_workspace_bytes(x.shape[0], tiles, most, inner)
    native.call("kudacuda_lora_add", x.data_ptr(), s["down"].data_ptr(), s["laid"].data_ptr(), s["ranks"].data_ptr(),
                s["scales"].data_ptr(), s["order"].data_ptr(), s["tiles"].data_ptr(), base.data_ptr(), out.data_ptr(),
                _workspace(nbytes).data_ptr(), nbytes, CODES[s["case"]["dtype"]], x.shape[0], tiles, adapters, most,
                inner, base.shape[1], x.stride(0), base.stride(0), out.stride(0),
                torch.cuda.current_stream().cuda_stream)
    return {"out": out}


def run(state) -> dict:
    kind = state["case"]["kind"]
    if own:
        return {"append": _own_append, "read": _own_read, "attention": _own_attention, "adapters": _own_adapters}[kind](state)
    return {"append": _plain_append, "read": _plain_read, "attention": _plain_attention,
            "adapters": _plain_adapters}[kind](state)


# ----------------------------------------------------------------- 64 bits
def exact(case, seed):
    """The cache's numbers, attention and adapted rows in 64 bits."""

    make = {"append": _exact_append, "read": _exact_read, "attention": _exact_attention, "adapters": _exact_adapters}
    return make[case["kind"]](prepare(case, seed))


def _exact_power(exponent) -> torch.Tensor:
    """2^exponent for whole exponents (a library's power may be off in the last place)."""

    return ((exponent.long() + 1023) << 52).view(torch.float64)


def _exact_values(case, pool, at, offset) -> torch.Tensor:
    """Rows (at, offset) of a pool from the fields of their bits: [rows, kv_heads, dim]."""

    elements, blocks = (part[at, :, offset].long() for part in _parts(case, pool))
    width, mantissa, bias = (4, 1, 1) if case["bits"] == 4 else (8, 3, 7)
    if width == 4:
        elements = torch.stack([elements % 16, elements // 16], dim=-1).flatten(-2)
    fraction = (elements % (1 << mantissa)).double() / (1 << mantissa)
    exponent = (elements >> mantissa) % (1 << (width - 1 - mantissa))
    size = torch.where(exponent > 0, (1 + fraction) * _exact_power(exponent - bias), fraction * 2.0 ** (1 - bias))
    size = torch.where(elements >> (width - 1) == 1, -size, size).unflatten(-1, (-1, BLOCK))
    power = torch.where(blocks > 0, _exact_power(blocks - 127), 0.0)
    return (size * power[..., None]).flatten(-2)


def _exact_read(s) -> dict:
    case, page = s["case"], s["case"]["page"]
    at, offset = s["slots"] // page, s["slots"] % page
    return {"keys": _exact_values(case, s["keys"], at, offset), "values": _exact_values(case, s["values"], at, offset)}


def _exact_append(s) -> dict:
    """Each pair as a complex number times its turn; a row's blocks in steps of its power of two."""

    case, dtype = s["case"], s["qkv"].dtype
    h, g, d, r = case["heads"], case["kv_heads"], case["dim"], case["rotary"]
    turn = torch.polar(torch.full((), case["factor"], dtype=torch.float64, device=DEV),
                       torch.outer(s["positions"].double(), s["freq"]))
    qkv = s["qkv"].double().view(-1, h + 2 * g, d)
    first = torch.arange(r // 2, device=DEV) * (2 if case["pairs"] else 1)
    second = first + (1 if case["pairs"] else r // 2)
    product = torch.complex(qkv[:, :h + g, first], qkv[:, :h + g, second]) * turn[:, None]
    rows = qkv[:, :h + g].clone()
    rows[:, :, first], rows[:, :, second] = product.real.clone(), product.imag.clone()
    keys, values = rows[:, h:].to(dtype).double(), qkv[:, h + g:]
    mantissa, lowest, limit = (1, 0, 7.0) if case["bits"] == 4 else (3, -6, 464.0)
    held = []
    for x in (keys, values):
        x = x.unflatten(-1, (-1, BLOCK))
        top = x.abs().amax(dim=-1, keepdim=True)
        power = torch.floor(torch.log2((top / limit).clamp(min=2.0**-300))) + 1
        power = torch.where(top < limit * _exact_power(power - 1), power - 1, power)  # (the logarithm's own rounding)
        power = torch.where(top >= limit * _exact_power(power), power + 1, power)
        power = _exact_power(power.clamp(min=LOWEST[case["dtype"], case["bits"]]))
        m = x / power
        binade = torch.floor(torch.log2(m.abs().clamp(min=2.0**lowest)))
        binade = torch.where(m.abs().clamp(min=2.0**lowest) < _exact_power(binade), binade - 1, binade)
        step = _exact_power(binade - mantissa)
        held.append((torch.round(m / step) * step * power).flatten(-2))
    return {"query": rows[:, :h].contiguous(), "keys": held[0], "values": held[1]}


def _exact_attention(s) -> dict:
    """Sequence by sequence and head by head."""

    case = s["case"]
    h, g, page = case["heads"], case["kv_heads"], case["page"]
    new, cached = _lengths(case)
    out = torch.empty(s["query"].shape, dtype=torch.float64, device=DEV)
    begin = 0
    for i, (n, c) in enumerate(zip(new, cached)):
        j = torch.arange(n + c, device=DEV)
        keys, values = (_exact_values(case, s[x], s["table"][i, j // page].long(), j % page) for x in ("keys", "values"))
        see = torch.ones((n, n + c), dtype=torch.bool, device=DEV).tril(c)
        for head in range(h):
            scores = (s["query"][begin:begin + n, head].double() @ keys[:, head // (h // g)].T) * s["scale"]
            out[begin:begin + n, head] = torch.softmax(scores.masked_fill(~see, -math.inf), dim=1) @ values[:, head // (h // g)]
        begin += n
    return {"out": out}


def _exact_adapters(s) -> dict:
    """Request by request."""

    case, out = s["case"], s["base"].double()
    begin = 0
    for i, n in enumerate(_numbers(case["chunks"])):
        if i < case["adapters"]:
            x = s["x"][begin:begin + n].double()
            out[begin:begin + n] += s["scales"][i].double() * (x @ s["down"][i].double().T) @ s["up"][i].double().T
        begin += n
    return {"out": out}
