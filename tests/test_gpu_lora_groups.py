"""GPU: adapters whose second product takes several groups of 256 outputs a block, against products in 64 bits."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from tests.test_gpu_lora import Round, _call

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16


def _cut(batch, rows):
    """The plan with tiles of up to ``rows`` rows."""

    table = batch.tiles.cpu().numpy()
    tiles = []
    for a in np.unique(table[:, 0]):
        first, n = table[table[:, 0] == a, 1].min(), table[table[:, 0] == a, 2].sum()
        tiles += [(a, first + i, min(rows, n - i)) for i in range(0, n, rows)]
    batch.tiles = torch.tensor(np.array(tiles), dtype=torch.int32, device=batch.tiles.device)
    batch.tile_count = len(tiles)


# What a block takes: tiles * ceil(out / 256) / 640 groups, an even number of them, where tiles have up to 16 rows and
# ranks up to 64, otherwise / 2048; at most 16.
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("tiles,rows,ranks,outer,groups", [
    (64, 1, (8, 16, 32, 64), 5000, 2),     # 20 columns of 256
    (64, 1, (8, 16, 32, 64), 10920, 4),    # 43: the last block's fourth group lies behind the outputs
    (64, 1, (16,), 10760, 4),              # 43, of the last 8 outputs
    (130, 3, (1, 40, 9), 5200, 4),         # 21: the last block has one group, and three behind the outputs
    (300, 1, (8, 24), 10920, 16),          # the most
    (300, 2, (8,), 4104, 6),               # 17, of the last 8 outputs
    (150, 1, (128, 70, 5), 10920, 3),      # ranks above 64: one set of operands
    (200, 2, (100,), 5200, 2),
    (70, 20, (16, 33), 15368, 2),          # tiles of more than 16 rows; 61
    (240, 17, (8,), 8200, 3),              # 33
    (66, 17, (128, 90), 16000, 2),
])
def test_matches_fp64(torch_gpu, native, dtype, tiles, rows, ranks, outer, groups):
    columns = -(-outer // 256)
    share = tiles * columns // (640 if rows <= 16 and max(ranks) <= 64 else 2048)
    assert groups == (min(share, 16) // 2 * 2 if rows <= 16 and max(ranks) <= 64 else min(share, 16))
    n = 10  # adapters, and requests without one
    of = [None if i % 11 == 10 else (i % 11, ranks[i % 11 % len(ranks)]) for i in range(tiles)]
    print(f"adapters of ranks {ranks}, {tiles} tiles of {rows} rows, 64 -> {outer}, {dtype}", flush=True)
    r = Round(native, 31, [rows] * tiles, of, 64, outer, dtype=dtype, spare=0)
    assert len(r.factors) == n
    _cut(r.batch, rows)
    assert r.batch.tile_count == tiles
    x, base = r.rows(r.x), r.rows(r.base)
    out = torch.full_like(base, 7.25)
    want, bound = r.want()
    r.pool.add(r.batch, x, base, out)
    assert (np.abs(out.cpu().double().numpy() - want) <= bound).all()
    assert torch.equal(base.cpu(), r.base)
    r.pool.add(r.batch, x, base)  # in place: the same
    assert torch.equal(base, out)
    _call(native, r, x, 0, out)
    r.check(out, base=False)
