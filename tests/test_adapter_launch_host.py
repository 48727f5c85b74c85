"""How much of an SM the adapters' kernels take, checked where no GPU is needed."""

from __future__ import annotations

import pytest

from kvforge_b200 import ops

SM_SHARED = 228 * 1024  # of which a CTA takes 1 KB besides what it asks for
CTA_MOST = 227 * 1024
TENSOR_COLUMNS, CTA_COLUMNS = 512, 128


@pytest.mark.parametrize("sections", [1, 2, 3, 4])
@pytest.mark.parametrize("rank", range(16, 129, 16))
def test_clusters_do_not_wait_for_one_anothers_tensor_memory(sections, rank):
    """No SM holds more CTAs of the kernel that makes the inner numbers of many rows than have room in its tensor memory: a CTA that waits for
    room keeps the CTAs of its cluster waiting, which hold theirs on other SMs."""
    if sections * rank > ops.ADAPTER_MAX_ROWS:
        pytest.skip("no such bank")
    for k in (8, 64, 72, 512, 520, 1024, 1032, 4096, 14336, 65536):
        taken = ops._fn("kvf_adapter_inner_bytes", "adapters")(sections, rank, k)
        assert 0 < taken <= CTA_MOST
        assert SM_SHARED // (taken + 1024) * CTA_COLUMNS <= TENSOR_COLUMNS, k
