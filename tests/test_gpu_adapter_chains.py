"""Adapters of a step one after another: banks that share the groups and what lies between the products, with dependent launches and
without, eager and replayed, at the row counts where the kernels change."""

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


def row_counts():
    from kvforge_b200 import ops

    return [ops.ADAPTER_MANY - 1, ops.ADAPTER_MANY, ops.ADAPTER_MANY + 200, 2 * ops.ADAPTER_MANY + 31]


@pytest.mark.parametrize("n", row_counts())
@pytest.mark.parametrize("wide", [False, True])
def test_banks_that_share_their_groups(ops, n, wide):
    """Products of the own kernel with adapters of other ranks, sections and widths behind each, every one in the buffers of the
    one before; replayed with other ids."""
    banks = [
        make(ops, 4, 136, (512, 640, 768), 16, torch.bfloat16), make(ops, 4, 264, (520,), 64, torch.bfloat16), make(ops, 4, 72, (512, 1024), 24, torch.bfloat16, alternating=True),
        make(ops, 4, 200, (256, 600), 128, torch.bfloat16), make(ops, 4, 1024, (128,), 48, torch.bfloat16, ranks=[48, 3, 0, 17]),
    ]  # fmt: skip
    ids = torch.full((n,), -1, dtype=torch.int32, device="cuda")
    groups = ops.AdapterGroups(n, 4, "cuda")
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    xs, ws, bases, outs = [], [], [], []
    for i, b in enumerate(banks):
        x, _ = inputs(n, b.k, b.n, torch.bfloat16, False, seed=i)
        w = (torch.randn(b.n, b.k, generator=torch.Generator(device="cuda").manual_seed(i), device="cuda") * b.k**-0.5).bfloat16()
        base = torch.empty(n, b.n, dtype=torch.bfloat16, device="cuda")
        ops.gemm_tcgen05(x, w, base, err=err)
        torch.cuda.synchronize()
        xs.append(x), ws.append(w), bases.append(base.float() if wide else base)
        outs.append(torch.empty_like(bases[-1]))
    made = [torch.empty_like(b) for b in bases]
    narrow = [torch.empty(n, b.n, dtype=torch.bfloat16, device="cuda") for b in banks]

    def step():
        ops.group_by_adapter(ids, groups, err)
        for i, bank in enumerate(banks):
            ops.gemm_tcgen05(xs[i], ws[i], narrow[i], err=err)
            if wide:
                made[i].copy_(narrow[i])
            else:
                made[i] = narrow[i]
            ops.adapter_add(xs[i], bank, groups, outs[i], base=made[i])
            ops.adapter_add(xs[i], bank, groups, made[i])  # and in place

    def check(chosen):
        torch.cuda.synchronize()
        for i, bank in enumerate(banks):
            want, mag = formula(xs[i], bank, chosen, bases[i])
            close(outs[i], want, mag, outs[i].dtype)
            close(made[i], want, mag, outs[i].dtype)
        assert int(err) == 0

    first = mixed_ids(n, 4, seed=9)
    ids.copy_(torch.tensor(first, dtype=torch.int32))
    step()
    check(first)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for turn in range(3):
        chosen = mixed_ids(n, 4, seed=turn) if turn < 2 else [i * 4 // n for i in range(n)]
        ids.copy_(torch.tensor(chosen, dtype=torch.int32))
        graph.replay()
        check(chosen)


def test_many_rows_of_a_bank_beyond_32_bits(ops):
    """The last adapter of a bank of more than 2^31 numbers, through the maps of the kernels of many rows."""
    s, k, n = 2400, 8192, 8192
    a = torch.zeros(s, 1, 128, k, dtype=torch.bfloat16, device="cuda")
    b = torch.zeros(s, n, 128, dtype=torch.bfloat16, device="cuda")
    a[s - 1] = torch.randn(1, 128, k, device="cuda") * k**-0.5
    b[s - 1] = torch.randn(n, 128, device="cuda")
    bank = ops.AdapterBank(a, b, torch.ones(s, device="cuda"))
    rows = ops.ADAPTER_MANY + 7
    for wide in (False, True):
        x, base = inputs(rows, k, n, torch.bfloat16, wide)
        ids = [s - 1] * rows
        t = torch.tensor(ids, dtype=torch.int32, device="cuda")
        groups = ops.AdapterGroups(rows, s, "cuda")
        ops.group_by_adapter(t, groups)
        out = torch.full_like(base, float("nan"))
        ops.adapter_add(x, bank, groups, out, base=base)
        want, mag = formula(x, bank, ids, base)
        close(out, want, mag, base.dtype)
