"""Calls of the entry points for caches of fewer bits and for adapters that must be refused before anything is launched."""

from __future__ import annotations

from tests._refusals import APPEND, ATTEND, P, Q

_PAGES = dict(num_pages=4, page_size=16, page_stride=2304)
MX_APPEND = {k: v for k, v in APPEND.items() if k not in ("page_stride", "head_stride", "token_stride", "amplitude", "stream")}
MX_APPEND = {k: v for name, value in MX_APPEND.items() for k, v in ([(name, value), ("bits", 4)] if name == "dtype" else
                                                                      [(name, value)])} | _PAGES | dict(amplitude=1.0, stream=0)
MX_READ = dict(key_pages=P, value_pages=P, slots=P, key_output=P, value_output=Q, dtype=1, bits=4, tokens=3, kv_heads=2,
               head_dim=128, key_stride=256, value_stride=256, **_PAGES, stream=0)
MX_ATTEND = {k: v for name, value in ATTEND.items() for k, v in ([(name, value), ("bits", 8)] if name == "dtype" else
                                                                   [(name, value)])
             if k not in ("page_stride", "head_stride", "token_stride", "scale", "stream")}
MX_ATTEND |= dict(page_stride=2112 + 64, scale=0.125, stream=0)
LORA = dict(input=P, a_factors=P, b_factors=P, ranks=P, scales=P, order=P, tiles=P, base=Q, output=Q, workspace=P,
            workspace_bytes=1 << 20, dtype=1, tokens=5, tile_count=2, adapters=3, max_rank=16, in_features=64,
            out_features=128, input_stride=64, base_stride=128, output_stride=128, stream=0)
CALLS = {"kudacuda_rope_paged_append_mx": MX_APPEND, "kudacuda_paged_read_mx": MX_READ,
         "kudacuda_paged_attention_mx": MX_ATTEND, "kudacuda_lora_add": LORA}

_PAGE_CHANGES = [
    (dict(bits=16), "bits"), (dict(bits=0), "bits"), (dict(head_dim=96), "head_dim"), (dict(kv_heads=0), "kv_heads"),
    (dict(num_pages=0), "num_pages"), (dict(num_pages=1 << 31), "num_pages"), (dict(page_size=8), "power of two"),
    (dict(page_size=24), "power of two"), (dict(page_size=8192), "power of two"), (dict(page_stride=2160), "page_stride"),
    (dict(page_stride=4100), "16-byte"), (dict(page_stride=1 << 31), "page_stride"), (dict(key_pages=P + 8), "16-byte"),
    (dict(value_pages=P + 4), "16-byte"), (dict(key_pages=0), "non-null"), (dict(dtype=0), "dtype")]
CHANGES = {
    "kudacuda_rope_paged_append_mx": _PAGE_CHANGES + [
        (dict(slots=0), "non-null"), (dict(tokens=-1), "tokens>=0"), (dict(query_heads=0), "heads"),
        (dict(rotary_dim=130), "rotary_dim"), (dict(interleaved=2), "interleaved"), (dict(key_stride=255), "strides"),
        (dict(value_stride=0), "strides"), (dict(query_stride=768), "in place"), (dict(slots=P + 4), "aligned"),
        (dict(inv_freq=P + 4), "aligned"), (dict(query=P + 1), "aligned"), (dict(amplitude=float("inf")), "amplitude"),
        (dict(tokens=1 << 26), "2^25")],
    "kudacuda_paged_read_mx": _PAGE_CHANGES + [
        (dict(slots=0), "non-null"), (dict(value_output=0), "non-null"), (dict(tokens=-1), "tokens"),
        (dict(tokens=(1 << 30) + 1), "2^30"), (dict(key_stride=255), "strides"), (dict(value_stride=260), "strides"),
        (dict(key_output=P + 8), "16-byte"), (dict(slots=P + 4), "16-byte"), (dict(key_output=Q), "two outputs")],
    "kudacuda_paged_attention_mx": [c for c in _PAGE_CHANGES if "page_stride" not in c[0]] + [
        (dict(page_stride=2096), "page_stride"), (dict(page_table=0), "non-null"), (dict(output=0), "non-null"),
        (dict(query_heads=5), "multiple of kv_heads"), (dict(query_heads=2048), "query_heads"), (dict(tokens=-1), "tokens"),
        (dict(sequences=0), "sequences"), (dict(sequences=65537), "sequences"), (dict(table_stride=0), "table_stride"),
        (dict(table_stride=1 << 27), "table_stride"), (dict(max_query_len=0), "max_query_len"),
        (dict(max_kv_len=0), "max_kv_len"), (dict(query_stride=252), "strides"), (dict(output_stride=260), "strides"),
        (dict(query=P + 8), "16-byte"), (dict(workspace=P + 4), "16-byte"), (dict(kv_lens=P + 2), "16-byte"),
        (dict(workspace_bytes=-1), "workspace_bytes"), (dict(scale=0.0), "scale"), (dict(scale=float("nan")), "scale"),
        (dict(output=P), "apart"), (dict(tokens=(1 << 25) + 1), "2^27"),
        (dict(sequences=65536, query_heads=128, kv_heads=128, page_stride=1 << 20), "2^22")],
    "kudacuda_lora_add": [
        (dict(input=0), "non-null"), (dict(tiles=0), "non-null"), (dict(output=0), "non-null"), (dict(dtype=0), "dtype"),
        (dict(tokens=-1), "tokens"), (dict(tokens=(1 << 20) + 1), "2^20"), (dict(adapters=0), "adapters"),
        (dict(adapters=65537), "adapters"), (dict(max_rank=12), "max_rank"), (dict(max_rank=136), "max_rank"),
        (dict(max_rank=0), "max_rank"), (dict(in_features=60), "in_features"), (dict(in_features=1 << 18), "in_features"),
        (dict(out_features=4), "out_features"), (dict(tile_count=-1), "tile_count"), (dict(tile_count=1 << 21), "2^31"),
        (dict(input_stride=56), "strides"), (dict(output_stride=120), "strides"), (dict(base_stride=132), "strides"),
        (dict(input=P + 8), "16-byte"), (dict(workspace=P + 8), "16-byte"), (dict(order=P + 2), "16-byte"),
        (dict(output=P, base=P), "apart"), (dict(base_stride=256), "in place"), (dict(workspace=0), "workspace"),
        (dict(workspace_bytes=100), "workspace")],
}


def addresses(name: str) -> list[str]:
    return [k for k, v in CALLS[name].items() if v in (P, Q) and k != "workspace_bytes"]


def refusals():
    """(entry point, arguments by name, part of the reason)"""

    for name, changes in CHANGES.items():
        for change, reason in changes:
            assert set(change) <= set(CALLS[name]), (name, change)
            yield name, CALLS[name] | change, reason
