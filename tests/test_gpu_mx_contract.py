"""GPU: what the entry points for caches of fewer bits say of pages that lie too far apart."""

from __future__ import annotations

import pytest

from tests._mx_refusals import CALLS

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name", ["kudacuda_rope_paged_append_mx", "kudacuda_paged_read_mx", "kudacuda_paged_attention_mx"])
@pytest.mark.parametrize("stride", [1 << 31, 1 << 40])
def test_pages_too_far_apart_are_refused_as_such(torch_gpu, native, name, stride):
    """(Refused on the host: no address of the call is used.)"""

    values = CALLS[name] | {"page_stride": stride}
    assert getattr(native.lib, name)(native.handle, *values.values()) == 1
    assert "page_stride below 2^31" in native.error()
