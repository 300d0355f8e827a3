"""Plain 64-bit forms of the paged-cache operators on the host (test infrastructure), and random inputs for them."""

from __future__ import annotations

import numpy as np
import torch

HALF = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}  # half a step, relative
CODE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def f64(x: torch.Tensor) -> np.ndarray:
    return x.detach().cpu().double().numpy()


# ------------------------------------------------------------------- rotary
def rope(x: np.ndarray, positions: np.ndarray, freq: np.ndarray, amplitude: float, pairs: bool) -> np.ndarray:
    """x [tokens, heads, dim] as fp64."""

    out = x.copy()
    half = len(freq)
    angle = positions.astype(np.float64)[:, None] * freq[None, :]
    cos, sin = np.cos(angle)[:, None] * amplitude, np.sin(angle)[:, None] * amplitude
    first = np.arange(half) * 2 if pairs else np.arange(half)
    second = first + 1 if pairs else first + half
    out[..., first] = x[..., first] * cos - x[..., second] * sin
    out[..., second] = x[..., first] * sin + x[..., second] * cos
    return out


def rope_bound(x: np.ndarray, want: np.ndarray, half: int, pairs: bool, amplitude: float, dtype) -> np.ndarray:
    """Half a step of the result's type, and the fp32 arithmetic: the reduced angle (|phi| < 0.79) is off by its own,
    pi / 2's and the product's rounding, 3 * 2^-25; the polynomials by four roundings of 2^-24 and a remainder below
    2^-29; the amplitude, its product, and the pair's product and sum by 2^-24 each: under 10 * 2^-24 < 2^-20 of
    (|x1| + |x2|) * amplitude.  (Results below the type's smallest normal number round by a fixed step: 2^-25.)"""

    sums = np.abs(x).copy()
    first = np.arange(half) * 2 if pairs else np.arange(half)
    second = first + 1 if pairs else first + half
    both = np.abs(x[..., first]) + np.abs(x[..., second])
    sums[..., first] = both
    sums[..., second] = both
    return HALF[dtype] * np.abs(want) + 2.0**-20 * sums * abs(amplitude) + 2.0**-25


# ---------------------------------------------------------------- attention
class Paged:
    """A ragged batch over a paged cache.  layout "hnd": [pages, heads, size, dim], "nhd": [pages, size, heads, dim]."""

    def __init__(self, seed, new, kv, *, heads=4, kv_heads=2, dim=64, page=16, dtype=torch.bfloat16, layout="hnd",
                 spare=0, extra_rows=0, scale=None, q_extra=0, junk=float("nan")):
        rng = np.random.default_rng([77, seed])
        self.new, self.kv, self.page, self.dtype, self.dim = list(new), list(kv), page, dtype, dim
        self.heads, self.kv_heads, self.layout = heads, kv_heads, layout
        self.hint = None  # the longest length that calls are told; the batch's if None
        self.scale = float(np.float32(dim**-0.5 if scale is None else scale))
        used = [-(-n // page) for n in kv]
        self.num_pages = sum(used) + 3 + spare
        order = rng.permutation(self.num_pages)
        # entries behind a sequence's pages are never valid ids
        self.table = np.full((len(kv), max(1, max(used))), -7, dtype=np.int32)
        at = 0
        for i, n in enumerate(used):
            self.table[i, :n] = order[at:at + n]
            at += n
        self.tokens = sum(new) + extra_rows
        self.starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)

        def normal(*shape):
            return torch.from_numpy(rng.standard_normal(shape).astype(np.float32))

        self.q = normal(self.tokens, heads, dim + q_extra).to(dtype)[..., :dim].contiguous()
        self.q_pitch = heads * dim + q_extra * 8
        shape = (self.num_pages, kv_heads, page, dim)
        self.k = (normal(*shape) * 1.5).to(dtype)
        self.v = normal(*shape).to(dtype)
        # rows that no sequence has hold anything
        live = np.zeros((self.num_pages, page), dtype=bool)
        for i, n in enumerate(kv):
            for j in range(n):
                live[self.table[i, j // page], j % page] = True
        dead = torch.from_numpy(~live)
        for x in (self.k, self.v):
            x.transpose(1, 2)[dead] = junk

    def rows(self, pool: np.ndarray, i: int, g: int) -> np.ndarray:
        j = np.arange(self.kv[i])
        return pool[self.table[i, j // self.page], g, j % self.page]

    def want(self):
        """(out, sum of |weight * value|) in fp64; rows of no sequence are NaN."""

        out = np.full((self.tokens, self.heads, self.dim), np.nan)
        size = out.copy()
        queries, keys, values = f64(self.q), f64(self.k), f64(self.v)
        for i, (n, kv) in enumerate(zip(self.new, self.kv)):
            pos = kv - n + np.arange(n)
            hidden = np.arange(kv)[None, :] > pos[:, None]
            for h in range(self.heads):
                g = h // (self.heads // self.kv_heads)
                k, v = self.rows(keys, i, g), self.rows(values, i, g)
                q = queries[self.starts[i]:self.starts[i] + n, h]
                with np.errstate(invalid="ignore"):
                    s = np.where(hidden, -np.inf, q @ k.T * self.scale) if kv else np.zeros((n, 0))
                top = s.max(axis=1, initial=-np.inf, keepdims=True)
                p = np.exp(s - np.where(np.isinf(top), 0.0, top))
                total = p.sum(axis=1, keepdims=True)
                p = np.divide(p, total, out=np.zeros_like(p), where=total > 0)
                at = slice(self.starts[i], self.starts[i] + n)
                if np.isfinite(v).all():
                    out[at, h], size[at, h] = p @ v, p @ np.abs(v)
                    continue
                for row in range(n):
                    seen = slice(0, max(0, min(kv, pos[row] + 1)))
                    out[at.start + row, h] = p[row, seen] @ v[seen]
                    size[at.start + row, h] = p[row, seen] @ np.abs(v[seen])
        return out, size

    def bound(self, want, size):
        """How far an output may be off: half a step of its type (and its smallest step, 2^-25 in fp16), half a step
        for each weight's rounding (relative to sum |weight * value|; an fp16 weight below 2^-14 rounds by up to
        2^-25 instead, of a maximum of 1, so every key adds at most that times its value), and the scores' fp32
        sums: at most dim * 2^-24 of sum |q k| * scale, which for these inputs is below 32 (a normal pair has
        sum |q k| * scale about 0.95 sqrt(dim) <= 11) -- exp turns that into a relative error of
        128 * 2^-24 * 32 = 2^-12 of a weight, as the sums of up to 2^12 weights again at most."""

        half = HALF[self.dtype]
        tiny = 2.0**-25 if self.dtype == torch.float16 else 0.0
        top = max(1.0, float(np.nanmax(np.abs(np.where(np.isfinite(size), size, 0.0)))))
        keys = max(self.kv + [1])
        return half * np.abs(want) + (half + 2.0**-11) * size + tiny * (1 + 4 * keys * top)

    # -------------------------------------------------------------- the call
    def device(self, extra_heads: int = 0):
        """Tensors on the GPU in this layout."""

        pitch = self.q_pitch
        q = torch.zeros((self.tokens, pitch), dtype=self.dtype, device="cuda:0")
        q[:, :self.heads * self.dim] = self.q.reshape(self.tokens, -1).cuda()
        k, v = self.k.cuda(), self.v.cuda()
        if self.layout == "nhd":
            k, v = k.transpose(1, 2).contiguous(), v.transpose(1, 2).contiguous()
            strides = (k.stride(0), k.stride(2), k.stride(1))
        else:
            strides = (k.stride(0), k.stride(1), k.stride(2))
        up = lambda a: torch.from_numpy(a).cuda()  # noqa: E731
        return dict(q=q, k=k, v=v, strides=strides, table=up(self.table), starts=up(self.starts),
                    lens=up(np.array(self.kv, dtype=np.int32)),
                    out=torch.full((self.tokens, self.heads, self.dim), 7.25, dtype=self.dtype, device="cuda:0"))

    def call(self, native, d, stream=None, workspace=None, max_new=None, max_kv=None, nbytes=None):
        max_new = max(1, max(self.new)) if max_new is None else max_new
        max_kv = (self.hint or max(1, max(self.kv))) if max_kv is None else max_kv
        n = len(self.new)
        if nbytes is None:
            nbytes = native.lib.kudacuda_paged_attention_workspace_bytes(self.tokens, n, max_new, max_kv, self.heads,
                                                                         self.kv_heads, self.dim)
        if workspace is None and nbytes > 0:
            workspace = torch.empty(nbytes, dtype=torch.uint8, device="cuda:0")
            d.setdefault("kept", []).append(workspace)
        stream = torch.cuda.current_stream() if stream is None else stream
        native.call("kudacuda_paged_attention", d["q"].data_ptr(), d["k"].data_ptr(), d["v"].data_ptr(),
                    d["table"].data_ptr(), d["starts"].data_ptr(), d["lens"].data_ptr(), d["out"].data_ptr(),
                    workspace.data_ptr() if nbytes > 0 else 0, nbytes, CODE[self.dtype], self.tokens, n, max_new, max_kv,
                    self.heads, self.kv_heads, self.dim, self.q_pitch, self.heads * self.dim, self.num_pages, self.page,
                    self.table.shape[1], *d["strides"], self.scale, stream.cuda_stream)
        return d["out"]


# ----------------------------------------------------------------- sampling
def sample(logits: np.ndarray, u: float, temperature: float, top_k: int, top_p: float, min_p: float):
    """(token, chance, distance): the definition in fp64 for one row, token by token down the order.  distance: how
    far u, and top_p, are from the place where another token would come out, relative to the sum."""

    x = np.where(np.isnan(logits), -np.inf, logits.astype(np.float64)) + 0.0
    order = np.argsort(-x, kind="stable")
    if not temperature > 0:
        return (0, 0.0, 1.0) if x[order[0]] == -np.inf else (int(order[0]), 1.0, 1.0)
    top = x[order[0]]
    if top == -np.inf:
        return 0, 0.0, 1.0
    with np.errstate(invalid="ignore"):
        w = np.where(x[order] == top, 1.0, np.exp((x[order] - top) / temperature))
    w[x[order] == -np.inf] = 0.0
    if 0 < top_k < len(w):
        w = w[:top_k]
    kept, distance = len(w), 1.0
    if top_p < 1.0:
        before = np.cumsum(w) - w
        target = top_p * w.sum()
        kept = int(np.count_nonzero(before < target))
        if top_p > 0.0:  # (otherwise nothing is before the target, whatever the weights' rounding)
            distance = min(distance, float(np.abs(before - target).min()) / w.sum())
    kept = max(1, min(kept, int(np.count_nonzero(w >= min(min_p, 1.0)))))
    ids, w = order[:kept], w[:kept]
    by_id = np.argsort(ids)
    ids, w = ids[by_id], w[by_id]
    edges = np.cumsum(w) / w.sum()
    at = min(int(np.searchsorted(edges, u, side="right")), kept - 1)
    while w[at] == 0.0:
        at -= 1
    distance = min(distance, float(np.abs(edges[:-1] - u).min(initial=1.0)))
    return int(ids[at]), float(w[at] / w.sum()), distance
