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


@pytest.mark.parametrize("hidden,inter,n", [(256, 1024, 1), (256, 1024, 3), (256, 1024, 16), (512, 4096, 600), (512, 8192, 260), (72, 400, 90)])
def test_rows_without_an_adapter_are_what_they_are_alone(hidden, inter, n):
    """Bit for bit, whoever the neighbours are: a few rows, many, and those of the library product."""
    ops, rt, part, _, _, x, ids = feed_forward(hidden, inter, 16, n)
    act, out = run(ops, rt, part, x, None)
    got_act, got_out = run(ops, rt, part, x, ids)
    none = (ids < 0).nonzero()[:, 0]
    same = torch.equal(got_act[none], act[none]), torch.equal(got_out[none], out[none])
    assert same == (True, True)
    beyond = torch.where(ids < 0, torch.full_like(ids, 2), ids)  # ids outside the bank are none (and are reported)
    with pytest.raises(RuntimeError, match="adapter outside the bank"):
        run(ops, rt, part, x, beyond)
    assert torch.equal(rt.buf("mlp.act", n, inter), got_act)


@pytest.mark.parametrize("hidden,inter,rank,n", [(256, 1024, 16, 7), (256, 1024, 40, 16), (512, 4096, 16, 600), (512, 8192, 24, 260), (512, 4096, 128, 531)])
def test_gates_and_ups_are_rounded_once(hidden, inter, rank, n):
    """What gates and ups are joined to, against 64 bits.  It is rounded to bfloat16 once, and so are, of many rows with an adapter, a gate and an
    up as they leave the product and again with the adapter added (a rounding is off by 2^-8 of the value: eight significant bits).  A gate and an up are
    sums in 32 bits: no chain of more than 64 roundings, 2^-18 of the absolute terms; the numbers between an adapter's products are exact to 2^-18 where 32
    bits come out and to 2^-17 else.  The exponential and the quotient of a gate of at most 16 are off by 2^-18 of themselves; the activation grows by 1.1 of a
    gate's error at most."""
    ops, rt, part, weights, lora, x, ids = feed_forward(hidden, inter, rank, n)
    few = n <= ops.SKINNY_USE_M
    assert few or ops.tcgen05_ok(x, part.w_gate_up)
    act, _ = run(ops, rt, part, x, ids)
    xd = x.double()
    half = torch.finfo(torch.bfloat16).eps / 2
    sums, errors = [], []
    for proj in ("gate_proj", "up_proj"):
        w = weights[f"{proj}.weight"].double()
        s, m = xd @ w.t(), xd.abs() @ w.t().abs()
        off = torch.zeros_like(s) if few else (ids >= 0).double()[:, None] * half * s.abs()
        for slot, made in enumerate(lora):
            a, b = (made[f"mlp.{proj}.lora_{k}.weight"].double() for k in "AB")
            own = (ids == slot).double()[:, None]
            s += own * 0.75 * ((xd @ a.t()) @ b.t())
            m += own * 0.75 * ((xd.abs() @ a.t().abs()) @ b.t().abs())
        if not few:
            off += (ids >= 0).double()[:, None] * half * s.abs()
        sums.append(s)
        errors.append(off * (1 + 2 * half) + 2.0**-16 * m)
    (gate, up), (eg, eu) = sums, errors
    assert float(gate.abs().max()) < 16
    silu = gate * torch.sigmoid(gate)
    want = silu * up
    before = 1.1 * eg * (up.abs() + eu) + silu.abs() * eu + 2.0**-18 * want.abs()
    bound = before + half * (want.abs() + before) + 2.0**-30
    off = float(((act.double() - want).abs() / bound).max())
    assert off <= 1.0
