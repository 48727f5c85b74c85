"""Float32 adapters, whose partial sums and columns take one another's place in shared memory."""

from __future__ import annotations

import pytest
import torch

from test_gpu_adapters import close, formula, inputs, make, mixed_ids

pytestmark = pytest.mark.gpu


@pytest.fixture(params=[False, True], ids=["plain", "dependent"])
def ops(request):
    from kvforge_b200 import ops as o

    before = bool(o._pdl_state)
    o.set_pdl(request.param)
    yield o
    o.set_pdl(before)


@pytest.mark.parametrize("n", [1, 5, 40, 90, 515])
@pytest.mark.parametrize("k,ends,rank", [(2048, (2048,), 16), (136, (512, 1024, 1536), 48), (4096, (264, 528), 128), (520, (96, 192, 288, 384), 32)])
def test_float32_sums_and_the_columns_that_take_their_place(ops, n, k, ends, rank):
    """Partial sums in shared memory, then columns of B and of the rows by bulk copies in the same place, section after section: the
    values, and the same bits every time."""
    bank = make(ops, 3, k, ends, rank, torch.float32)
    x, base = inputs(n, k, ends[-1], torch.float32, True)
    ids = mixed_ids(n, 3)
    groups = ops.AdapterGroups(n, 3, "cuda")
    ops.group_by_adapter(torch.tensor(ids, dtype=torch.int32, device="cuda"), groups)
    want, mag = formula(x, bank, ids, base)
    outs = [torch.full_like(base, float("nan")) for _ in range(20)]
    for out in outs:
        ops.adapter_add(x, bank, groups, out, base=base)
    close(outs[0], want, mag, torch.float32)
    assert all(torch.equal(o, outs[0]) for o in outs)
