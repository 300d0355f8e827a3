"""Calls of the paged-cache entry points that must be refused before anything is launched."""

from __future__ import annotations

import numpy as np

P = 1 << 20  # 16-byte aligned addresses that are never read: every call below is refused
Q = P + (1 << 19)
ROPE = dict(input=P, inv_freq=P, positions=P, output=P, dtype=1, tokens=3, heads=2, head_dim=128, rotary_dim=128,
            interleaved=0, input_stride=256, output_stride=256, amplitude=1.0, stream=0)
APPEND = dict(query=P, key=P, value=P, inv_freq=P, positions=P, slots=P, query_output=P, key_pages=P, value_pages=P,
              dtype=1, tokens=3, query_heads=4, kv_heads=2, head_dim=128, rotary_dim=64, interleaved=1,
              query_stride=512, key_stride=256, value_stride=256, output_stride=512, num_pages=4, page_size=16,
              page_stride=4096, head_stride=2048, token_stride=128, amplitude=1.0, stream=0)
ATTEND = dict(query=P, key_pages=P, value_pages=P, page_table=P, query_starts=P, kv_lens=P, output=Q, workspace=P,
              workspace_bytes=1 << 20, dtype=2, tokens=3, sequences=2, max_query_len=2, max_kv_len=50, query_heads=4,
              kv_heads=2, head_dim=64, query_stride=256, output_stride=256, num_pages=4, page_size=16, table_stride=4,
              page_stride=2048, head_stride=1024, token_stride=64, scale=0.125, stream=0)
COPY = dict(pool=P, pairs=0, count=0, pools=2, num_pages=8, page_bytes=256, page_stride=256, pool_stride=2048, stream=0)
SAMPLE = dict(logits=P, random=P, temperature=P, top_k=P, top_p=P, min_p=P, tokens_out=P, chances=P, workspace=P,
              workspace_bytes=1 << 20, dtype=1, rows=2, vocab=1000, stride=1000, stream=0)
CALLS = {"kudacuda_rope": ROPE, "kudacuda_rope_paged_append": APPEND, "kudacuda_paged_attention": ATTEND,
         "kudacuda_copy_pages": COPY, "kudacuda_sample_tokens": SAMPLE}

# entry point -> what changes in its call above, and a part of the reason it must give
CHANGES = {
    "kudacuda_rope": [
        (dict(input=0), "non-null"), (dict(positions=0), "non-null"), (dict(dtype=0), "dtype"),
        (dict(tokens=-1), "tokens>=0"), (dict(heads=0), "heads"), (dict(head_dim=127), "even head_dim"),
        (dict(head_dim=258), "even head_dim"), (dict(rotary_dim=0), "rotary_dim"), (dict(rotary_dim=130), "rotary_dim"),
        (dict(rotary_dim=3), "rotary_dim"), (dict(interleaved=2), "interleaved"), (dict(input_stride=255), "strides"),
        (dict(output_stride=-256), "strides"), (dict(amplitude=float("nan")), "amplitude"),
        (dict(inv_freq=P + 4), "aligned"), (dict(input=P + 1), "aligned"), (dict(tokens=(1 << 25) + 1), "2^25"),
        (dict(output_stride=512), "in place")],
    "kudacuda_rope_paged_append": [
        (dict(slots=0), "non-null"), (dict(value_pages=0), "non-null"), (dict(kv_heads=0), "kv_heads"),
        (dict(num_pages=0), "num_pages"), (dict(page_size=24), "power of two"), (dict(page_size=8192), "power of two"),
        (dict(key_stride=255), "strides"), (dict(value_stride=0), "strides"), (dict(token_stride=64), "pool strides"),
        (dict(page_stride=-4096), "pool strides"), (dict(slots=P + 4), "aligned"), (dict(dtype=3), "dtype"),
        (dict(query_stride=768), "in place"), (dict(tokens=1 << 26), "2^25")],
    "kudacuda_paged_attention": [
        (dict(page_table=0), "non-null"), (dict(output=0), "non-null"), (dict(dtype=0), "dtype"),
        (dict(head_dim=96), "head_dim"), (dict(query_heads=5), "multiple of kv_heads"), (dict(kv_heads=0), "kv_heads"),
        (dict(query_heads=2048, kv_heads=2048), "query_heads"), (dict(tokens=-1), "tokens"),
        (dict(tokens=1 << 29), "2^30"), (dict(sequences=0), "sequences"), (dict(sequences=65537), "sequences"),
        (dict(num_pages=0), "num_pages"), (dict(page_size=3), "power of two"), (dict(table_stride=0), "table_stride"),
        (dict(table_stride=1 << 27), "table_stride"), (dict(max_query_len=0), "max_query_len"),
        (dict(max_kv_len=0), "max_kv_len"), (dict(query_stride=252), "strides"), (dict(token_stride=68), "strides"),
        (dict(head_stride=0), "strides"), (dict(query=P + 8), "16-byte"), (dict(workspace=P + 4), "16-byte"),
        (dict(kv_lens=P + 2), "16-byte"), (dict(workspace_bytes=-1), "workspace_bytes"), (dict(scale=0.0), "scale"),
        (dict(output=P), "apart"), (dict(tokens=(1 << 25) + 1), "2^27"),
        (dict(sequences=65536, query_heads=128, kv_heads=128), "2^22"),
        (dict(scale=float("inf")), "scale"), (dict(scale=-1.0), "scale")],
    "kudacuda_copy_pages": [
        (dict(pool=0), "non-null"), (dict(count=1), "non-null"), (dict(count=-1), "count"), (dict(pools=0), "pools"),
        (dict(num_pages=0), "num_pages"), (dict(page_bytes=0), "page_bytes"), (dict(page_bytes=24), "16-byte"),
        (dict(pool=P + 8), "16-byte"), (dict(page_stride=240), "page_bytes"), (dict(pool_stride=128), "page_bytes"),
        (dict(pool_stride=256), "each other's"), (dict(pool_stride=1024), "each other's"),
        (dict(pairs=[(0, 8)]), "page ids"), (dict(pairs=[(-1, 2)]), "page ids"),
        (dict(pairs=[(0, 2), (1, 2)]), "differ"), (dict(pairs=[(0, 2), (2, 2)]), "differ"),
        (dict(pairs=[(0, 2), (2, 3)]), "source"), (dict(pairs=[(2, 3), (0, 2)]), "source"),
        (dict(pairs=[(0, 1), (1, 0)]), "source"), (dict(pairs=[(i, (i + 1) % 8) for i in range(8)]), "source"),
        (dict(pairs=[(0, 1)] * 9), "count"), (dict(pools=65536, page_bytes=1 << 22), "2^37")],
    "kudacuda_sample_tokens": [
        (dict(logits=0), "non-null"), (dict(random=0), "non-null"), (dict(tokens_out=0), "non-null"),
        (dict(workspace=0), "non-null"), (dict(dtype=3), "dtype"), (dict(rows=65536), "rows"), (dict(rows=-1), "rows"),
        (dict(vocab=0), "vocab"), (dict(vocab=(1 << 20) + 1, stride=1 << 21), "vocab"), (dict(stride=999), "stride"),
        (dict(workspace_bytes=1000), "workspace"), (dict(workspace=P + 8), "16-byte"), (dict(logits=P + 1), "aligned"),
        (dict(top_p=P + 2), "aligned")],
}
_kept: list[np.ndarray] = []


def _pairs(values: dict) -> dict:
    if isinstance(values["pairs"], list):
        table = np.ascontiguousarray(values["pairs"], dtype=np.int32).reshape(-1, 2)
        _kept.append(table)
        values = values | {"pairs": table.ctypes.data, "count": len(table)}
    return values


def refusals():
    """(entry point, arguments, part of the reason)"""

    for name, changes in CHANGES.items():
        for change, reason in changes:
            assert set(change) <= set(CALLS[name]), (name, change)
            values = CALLS[name] | change
            values = _pairs(values) if name == "kudacuda_copy_pages" else values
            yield name, tuple(values.values()), reason


def accepted():
    """The calls that the changes start from (their addresses are none: never made on a GPU)."""

    for name, values in CALLS.items():
        values = _pairs(values | {"pairs": [(0, 2), (1, 3), (4, 4), (4, 5)]}) if name == "kudacuda_copy_pages" else values
        yield name, tuple(values.values())
