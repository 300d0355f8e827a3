"""CPU: the workspaces of adapters' calls, which all adapters of a handle share stream by stream."""

from __future__ import annotations

import contextlib
from types import SimpleNamespace

import pytest
import torch

from kudacuda_amd.lora import LoraAdapters, lora_batch


class FakeCuda:
    """torch.cuda with a current stream, captured or not."""

    stream, capturing = 100, False

    def current_device(self):
        return 0

    def current_stream(self, device):
        return SimpleNamespace(cuda_stream=self.stream)

    def is_current_stream_capturing(self):
        return self.capturing

    @contextlib.contextmanager
    def device(self, device):
        yield


@pytest.fixture
def program():
    """Three projections' adapters (their tensors on the CPU), the fake torch.cuda and the calls that reach the library."""

    calls, cuda = [], FakeCuda()
    lib = SimpleNamespace(kudacuda_lora_workspace_bytes=lambda tokens, tiles, rank, inner: tokens * rank * 4)
    native = SimpleNamespace(call=lambda name, *args: calls.append(args), lib=lib, workspaces={})
    fake = SimpleNamespace(**{n: getattr(torch, n) for n in ("zeros", "empty", "bfloat16", "float16", "float32", "int32", "uint8",
                                                             "device")}, cuda=cuda)
    pools = [LoraAdapters(native, fake, in_features=8, out_features=8, adapters=1, max_rank=r, device="cpu") for r in (8, 32, 16)]
    batch = lora_batch(torch, [0], [4], device="cpu")
    batch.stream = 100
    rows = torch.zeros((4, 8), dtype=torch.bfloat16), torch.zeros((4, 8), dtype=torch.bfloat16)
    return native, cuda, pools, lambda pool: pool.add(batch, *rows), calls


def test_adapters_of_a_handle_share_one_workspace_a_stream(program):
    native, cuda, pools, add, calls = program
    for pool in (*pools, *pools):
        add(pool)
    assert [w.numel() for w in native.workspaces.values()] == [4 * 32 * 4]
    (kept,) = native.workspaces.values()
    assert {args[9] for args in calls[1:]} == {kept.data_ptr()} and [args[10] for args in calls[:3]] == [128, 512, 256]


def test_another_stream_and_a_captured_call_have_their_own(program):
    native, cuda, pools, add, calls = program
    add(pools[1])
    cuda.capturing = True
    add(pools[0])
    assert len(native.workspaces) == 1 and calls[0][9] != calls[1][9]
    cuda.capturing = False
    lora = pools[0]
    cuda.stream = 200
    batch = lora_batch(torch, [0], [4], device="cpu")
    batch.stream = 200
    lora.add(batch, torch.zeros((4, 8), dtype=torch.bfloat16), torch.zeros((4, 8), dtype=torch.bfloat16))
    assert len({w.data_ptr() for w in native.workspaces.values()}) == 2 and calls[2][9] != calls[0][9]
