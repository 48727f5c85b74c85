"""A gated feed-forward in steps with low-rank adapters: which product runs, and what is rounded."""

from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

pytestmark = pytest.mark.gpu


def feed_forward(hidden, inter, rank, n, seed=0):
    """A gated feed-forward with two adapters, a step's rows, and every third row without an adapter."""
    from kvforge_b200 import ops
    from kvforge_b200.engine.runtime import Runtime
    from kvforge_b200.parts.adapters import AdapterStore
    from kvforge_b200.parts.mlp import GatedMLP

    g = torch.Generator(device="cuda").manual_seed(seed + n)
    normal = lambda *shape, s: (torch.randn(*shape, generator=g, device="cuda") * s).bfloat16()  # noqa: E731
    rt = Runtime("cuda", torch.bfloat16, max(n, 16), 16)
    rt.adapters = AdapterStore(2, rank, max(n, 16), torch.bfloat16, torch.device("cuda"))
    part = GatedMLP({"hidden_size": hidden, "intermediate_size": inter}, prefix="mlp.")
    weights = {
        "gate_proj.weight": normal(inter, hidden, s=hidden**-0.5), "up_proj.weight": normal(inter, hidden, s=hidden**-0.5),
        "down_proj.weight": normal(hidden, inter, s=inter**-0.5),
    }  # fmt: skip
    part.bind(weights, rt)
    names = part.gate_up_bank, part.down_bank
    lora = []
    for slot in range(2):
        made = {}
        for d in rt.adapters._declared:
            for proj, width in zip(d.names, d.widths):
                made[f"{proj}.lora_A.weight"] = normal(rank, d.bank.k, s=d.bank.k**-0.5)
                made[f"{proj}.lora_B.weight"] = normal(width, rank, s=rank**-0.5)
        rt.adapters.load(f"a{slot}", made, 0.75)
        lora.append(made)
    assert all(names)
    x = normal(n, hidden, s=1.0)
    ids = torch.tensor([i % 3 - 1 for i in range(n)], dtype=torch.int32, device="cuda")
    return ops, rt, part, weights, lora, x, ids


def run(ops, rt, part, x, ids):
    """(what the gates and ups are joined to, the result) of a step, with adapters where ``ids`` are given."""
    n = x.shape[0]
    ctx = SimpleNamespace(adapters=None, residual=torch.zeros(n, part.hidden, device="cuda"))
    if ids is not None:
        ctx.adapters = rt.adapters.groups
        ops.group_by_adapter(ids, ctx.adapters, rt.err)
    y = part.forward(ctx, x)
    out = ctx.residual if y is ops.ADDED else y.t.sum(0) if isinstance(y, ops.Partials) else y
    rt.check_error_flag()
    return rt.buf("mlp.act", n, part.inter).clone(), out.clone()


def test_gates_and_ups_of_many_rows_do_not_leave_the_own_kernel(monkeypatch):
    """The product that runs without adapters runs with them too: no library product takes its place."""
    ops, rt, part, _, _, x, ids = feed_forward(512, 4096, 16, 600)
    taken = []
    plain = ops.linear
    monkeypatch.setattr(ops, "linear", lambda a, w, out: (taken.append(w.data_ptr()), plain(a, w, out)))
    run(ops, rt, part, x, ids)
    assert part.w_gate_up.data_ptr() not in taken
