"""GPU: attention over 4- and 8-bit pages, single tokens with a long past beside prompts and chunks."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from tests._mx_ref import MxPaged
from tests._paged_ref import f64

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("new,kv,heads,kv_heads", [
    ([1000, 1, 1], [1000, 5000, 40], 16, 16), ([1, 300, 300, 2], [6000, 300, 900, 3000], 24, 12),
    ([700, 0, 1, 1], [1400, 9, 4000, 0], 16, 16)])
def test_matches_fp64(torch_gpu, native, dtype, bits, dim, new, kv, heads, kv_heads):
    batch = MxPaged(24, new, kv, bits=bits, heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype)
    print(f"attention in {bits} bits, {new} of {kv}, {heads}/{kv_heads} heads of {dim}", flush=True)
    d = batch.device()
    want, size = batch.want()
    for nbytes in (None, 0):
        got = f64(batch.call(native, d, nbytes=nbytes))
        assert np.isfinite(got).all()
        assert (np.abs(got - want) <= batch.bound(want, size)).all()
