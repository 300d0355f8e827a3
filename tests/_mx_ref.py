"""Plain host forms of the microscaled cache's numbers, and ragged batches over it (test infrastructure)."""

from __future__ import annotations

import numpy as np
import torch

from tests._paged_ref import CODE, Paged

BLOCK = 32


def levels(bits: int) -> np.ndarray:
    """What the codes of an element stand for, by code."""

    width, mantissa, bias = (4, 1, 1) if bits == 4 else (8, 3, 7)
    out = np.zeros(1 << width)
    for code in range(1 << width):
        fraction, exponent = code % (1 << mantissa), (code >> mantissa) % (1 << (width - 1 - mantissa))
        size = fraction * 2.0 ** (1 - bias - mantissa) if exponent == 0 else (1 + fraction / 2**mantissa) * 2.0 ** (exponent - bias)
        if bits == 8 and code % 128 == 127:
            size = np.nan
        out[code] = -size if code >> (width - 1) else size
    return out


def exponents(bits: int, dtype) -> tuple[int, int]:
    """The least and the greatest exponent of a block that is written."""

    if dtype == torch.bfloat16:
        return -110, 125 if bits == 4 else 119
    return (-23, 13) if bits == 4 else (-15, 7)


def pack(x: np.ndarray, bits: int, dtype) -> tuple[np.ndarray, np.ndarray]:
    """x [..., dim] (numbers of the type, in fp64) as codes [..., dim] and blocks' bytes [..., dim / 32], by trying the
    exponents from below and taking the nearest level, of two the even code."""

    x = x.reshape(*x.shape[:-1], -1, BLOCK)
    with np.errstate(invalid="ignore"):
        top = np.abs(x).max(axis=-1)
    limit = 7.0 if bits == 4 else 464.0
    low, high = exponents(bits, dtype)
    finite = np.isfinite(top)
    e = np.full(top.shape, low)
    sizes = np.log2(top[finite & (top > 0)]) if (finite & (top > 0)).any() else np.zeros(1)
    for exponent in range(max(low, int(sizes.min()) - 12), min(high, int(sizes.max()) + 2)):
        with np.errstate(invalid="ignore"):
            e[finite & (top >= limit * 2.0**exponent)] = exponent + 1
    table = levels(bits)
    positive = table[:(8 if bits == 4 else 127)]
    m = np.abs(np.where(finite[..., None], x, 0.0)) / (2.0 ** e.astype(np.float64))[..., None]
    above = np.clip(np.searchsorted(positive, m), 0, len(positive) - 1)
    below = np.maximum(above - 1, 0)
    to_above, to_below = positive[above] - m, m - positive[below]
    code = np.where((to_above < to_below) | ((to_above == to_below) & (above % 2 == 0)) | (to_above <= 0), above, below)
    code = code + np.where(np.signbit(x) & finite[..., None], 1 << (bits - 1), 0)
    return code.reshape(*code.shape[:-2], -1).astype(np.uint8), np.where(finite, e + 127, 255).astype(np.uint8)


def unpack(codes: np.ndarray, blocks: np.ndarray, bits: int) -> np.ndarray:
    power = np.where(blocks == 255, np.nan, 2.0 ** (blocks.astype(np.float64) - 127))
    x = levels(bits)[codes]
    return (x.reshape(*x.shape[:-1], -1, BLOCK) * power[..., None]).reshape(x.shape)


def to_bytes(codes: np.ndarray, bits: int) -> np.ndarray:
    return codes[..., 0::2] | codes[..., 1::2] << 4 if bits == 4 else codes


def to_codes(data: np.ndarray, bits: int) -> np.ndarray:
    return np.stack([data & 15, data >> 4], axis=-1).reshape(*data.shape[:-1], -1) if bits == 4 else data


def page_bytes(kv_heads: int, page: int, dim: int, bits: int) -> int:
    return kv_heads * page * (dim * bits // 8 + dim // BLOCK)


def to_pages(codes: np.ndarray, blocks: np.ndarray, bits: int, extra: int = 0) -> np.ndarray:
    """codes [pages, kv_heads, page, dim] and blocks as pages of bytes, ``extra`` of 0xa5 behind each."""

    pages = codes.shape[0]
    parts = [to_bytes(codes, bits).reshape(pages, -1), blocks.reshape(pages, -1)]
    return np.concatenate(parts + [np.full((pages, extra), 0xa5, dtype=np.uint8)], axis=1)


def from_pages(data: np.ndarray, kv_heads: int, page: int, dim: int, bits: int) -> tuple[np.ndarray, np.ndarray]:
    row = dim * bits // 8
    codes = to_codes(data[:, :kv_heads * page * row].reshape(-1, kv_heads, page, row), bits)
    at = kv_heads * page * row
    return codes, data[:, at:at + kv_heads * page * (dim // BLOCK)].reshape(-1, kv_heads, page, dim // BLOCK)


def numbers(x: np.ndarray, dtype) -> torch.Tensor:
    """fp64 numbers of the type as its tensor."""

    t = torch.from_numpy(np.ascontiguousarray(x)).to(dtype)
    assert torch.equal(t.double().nan_to_num(7.0), torch.from_numpy(np.ascontiguousarray(x)).nan_to_num(7.0))
    return t


class MxPaged(Paged):
    """A ragged batch over a cache of ``bits`` bits: k and v are what its pages hold."""

    def __init__(self, seed, new, kv, *, bits, page=16, extra=0, **kw):
        super().__init__(seed, new, kv, page=page, **kw)
        self.bits, self.extra = bits, extra
        self.repack()

    def repack(self) -> None:
        """The pages of k and v, and k and v what they hold."""

        self.pages = []
        for name in ("k", "v"):
            codes, blocks = pack(getattr(self, name).double().numpy(), self.bits, self.dtype)
            codes[np.repeat(blocks == 255, BLOCK, axis=-1)] = (1 << self.bits) - 2  # (anything)
            self.pages.append(to_pages(codes, blocks, self.bits, self.extra))
            setattr(self, name, numbers(unpack(codes, blocks, self.bits), self.dtype))

    def device(self, extra_heads: int = 0):
        d = super().device()
        d["k"], d["v"] = (torch.from_numpy(p).cuda() for p in self.pages)
        d["stride"] = d["k"].stride(0)
        return d

    def workspace_bytes(self, native, max_new=None, max_kv=None) -> int:
        return native.lib.kudacuda_paged_attention_mx_workspace_bytes(
            self.bits, self.tokens, len(self.new), max(1, max(self.new)) if max_new is None else max_new,
            (self.hint or max(1, max(self.kv))) if max_kv is None else max_kv, self.heads, self.kv_heads, self.dim)

    def call(self, native, d, stream=None, workspace=None, max_new=None, max_kv=None, nbytes=None):
        nbytes = self.workspace_bytes(native, max_new, max_kv) if nbytes is None else nbytes
        max_new = max(1, max(self.new)) if max_new is None else max_new
        max_kv = (self.hint or max(1, max(self.kv))) if max_kv is None else max_kv
        if workspace is None and nbytes > 0:
            workspace = torch.empty(nbytes, dtype=torch.uint8, device="cuda:0")
            d.setdefault("kept", []).append(workspace)
        stream = torch.cuda.current_stream() if stream is None else stream
        native.call("kudacuda_paged_attention_mx", d["q"].data_ptr(), d["k"].data_ptr(), d["v"].data_ptr(),
                    d["table"].data_ptr(), d["starts"].data_ptr(), d["lens"].data_ptr(), d["out"].data_ptr(),
                    workspace.data_ptr() if nbytes > 0 else 0, nbytes, CODE[self.dtype], self.bits, self.tokens,
                    len(self.new), max_new, max_kv, self.heads, self.kv_heads, self.dim, self.q_pitch,
                    self.heads * self.dim, self.num_pages, self.page, self.table.shape[1], d["stride"], self.scale,
                    stream.cuda_stream)
        return d["out"]
