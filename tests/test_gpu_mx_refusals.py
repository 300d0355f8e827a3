"""GPU: refusals of the entry points for caches of fewer bits and for adapters."""

from __future__ import annotations

import pytest
import torch

from tests import _mx_refusals
from tests._refusals import P

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name", list(_mx_refusals.CALLS))
def test_refusals_leave_a_reason(torch_gpu, native, name):
    buffer = torch.zeros(1 << 22, dtype=torch.uint8, device="cuda:0")
    for call, values, reason in _mx_refusals.refusals():
        if call == name:
            values = values | {k: buffer.data_ptr() + values[k] - P for k in _mx_refusals.addresses(name) if values[k] != 0}
            status = getattr(native.lib, call)(native.handle, *values.values())
            assert status == 1 and reason in native.error(), (call, values, native.error())
    torch.cuda.synchronize()
    assert int(buffer.count_nonzero()) == 0


@pytest.mark.parametrize("name", list(_mx_refusals.CALLS))
def test_no_tokens_is_a_call_that_does_nothing(torch_gpu, native, name):
    values = _mx_refusals.CALLS[name] | {"tokens": 0}
    assert getattr(native.lib, name)(native.handle, *values.values()) == 0, native.error()


def test_workspace_sizes_of_calls_that_are_refused(torch_gpu, native):
    lib = native.lib
    assert lib.kudacuda_paged_attention_mx_workspace_bytes(4, 1, 1, 1, 50000, 16, 2, 128) > 0
    for bad in ((5, 1, 1, 1, 50000, 16, 2, 128), (4, 0, 1, 1, 50000, 16, 2, 128), (4, 1, 1, 1, 50000, 16, 3, 128),
                (4, 1, 1, 1, 50000, 16, 2, 96)):
        assert lib.kudacuda_paged_attention_mx_workspace_bytes(*bad) == 0
    assert lib.kudacuda_lora_workspace_bytes(1, 1, 16, 2048) > 0
    for bad in ((0, 1, 16, 2048), (1, -1, 16, 2048), (1, 1, 12, 2048), (1, 1, 16, 0), (1 << 21, 1, 16, 2048)):
        assert lib.kudacuda_lora_workspace_bytes(*bad) == 0
