"""CPU: what the plan of attention over 4- and 8-bit pages makes of a batch, told by the workspace that it asks for."""

from __future__ import annotations

import pytest

from kudacuda_amd._native import load_library


@pytest.fixture(scope="module")
def splits():
    lib = load_library()

    def of(new, kv, heads, kv_heads, dim):
        """Partials that a row and head has room for."""

        tokens = sum(new)
        nbytes = lib.kudacuda_paged_attention_mx_workspace_bytes(4, tokens, len(new), max(new), max(kv), heads, kv_heads, dim)
        return nbytes // (tokens * heads * (dim + 2) * 4)

    return of


@pytest.mark.parametrize("new,kv,heads,kv_heads,dim", [
    ([2000, 1], [2000, 6001], 16, 2, 128), ([1500] + [1] * 8, [1500] + [1001 * i for i in range(1, 9)], 12, 4, 64),
    ([500, 500, 500, 1], [500, 500, 500, 8001], 12, 4, 64)])
def test_a_token_with_a_long_past_is_split_beside_a_prompt(splits, new, kv, heads, kv_heads, dim):
    """Its keys are shared by more blocks than the few that a prompt's tiles are split into."""

    assert splits(new, kv, heads, kv_heads, dim) >= 16


def test_chunks_behind_a_past_and_whole_prompts(splits):
    assert 2 <= splits([1200], [3200], 16, 2, 128) <= 8
    assert splits([2000], [2000], 16, 2, 128) <= 1
