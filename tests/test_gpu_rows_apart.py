"""Rows that leave the gated product before its activation, and the activation of single rows."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from kvforge_b200 import ops as o

    return o


def inputs(m, k, n, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + m * 3 + k + n)
    x = torch.randn(m, k, generator=g, device="cuda").bfloat16()
    w = (torch.randn(n, k, generator=g, device="cuda") * k**-0.5).bfloat16()
    ids = torch.randint(-2, 5, (m,), generator=g, device="cuda", dtype=torch.int32)
    return x, w, ids


@pytest.mark.parametrize("m,k,n", [(1, 8, 16), (7, 72, 48), (130, 64, 256), (300, 200, 528), (129, 1000, 4112)])
def test_rows_apart_are_those_of_the_two_products(ops, m, k, n):
    """Bit for bit: the plain product's rows and the gated product's rows; what belongs to neither stays."""
    x, w, ids = inputs(m, k, n)
    plain, gated = torch.empty(m, n, device="cuda", dtype=torch.bfloat16), torch.empty(m, n // 2, device="cuda", dtype=torch.bfloat16)
    ops.gemm_tcgen05(x, w, plain)
    ops.gemm_tcgen05(x, w, gated, mode="silu")
    store = torch.full((m, n + 8), 7.0, device="cuda", dtype=torch.bfloat16)
    out = torch.full_like(gated, 5.0)
    for count in (0, 1, 3, 100):
        store.fill_(7.0)
        out.fill_(5.0)
        ops.gemm_tcgen05(x, w, out, mode="silu", apart=(ids, count, store[:, :n]))
        taken = ((ids >= 0) & (ids < count))[:, None]
        assert torch.equal(out, torch.where(taken, torch.full_like(out, 5.0), gated))
        assert torch.equal(store[:, :n], torch.where(taken, plain, torch.full_like(plain, 7.0)))
        assert bool((store[:, n:] == 7).all())
        # and joined afterwards, those rows alone
        rows = store[:, :n].contiguous()
        whole = torch.empty_like(out)
        ops.silu_mul(plain, whole, interleaved=True)
        ops.silu_mul(rows, out, interleaved=True, rows=(ids, count))
        assert torch.equal(out, torch.where(taken, whole, gated))


@pytest.mark.parametrize("n,i,interleaved", [(1, 8, True), (5, 40, True), (5, 40, False), (300, 1032, True)])
def test_float_gates_and_ups_to_bfloat16(ops, n, i, interleaved):
    """One rounding (2^-8 of the value), and a float exponential, sum, quotient and product: 2^-18 for gates of at most 16."""
    g = torch.Generator(device="cuda").manual_seed(i)
    gu = (3 * torch.randn(n, 2 * i, generator=g, device="cuda")).clamp(-16, 16)
    out = torch.empty(n, i, device="cuda", dtype=torch.bfloat16)
    ops.silu_mul(gu, out, interleaved=interleaved)
    d = gu.double()
    gate, up = (d.view(n, -1, 2, 8)[:, :, k].reshape(n, i) for k in (0, 1)) if interleaved else (d[:, :i], d[:, i:])
    want = gate * torch.sigmoid(gate) * up
    assert bool(((out.double() - want).abs() <= want.abs() * (2.0**-8 + 2.0**-18) + 2.0**-120).all())


def test_refusals(ops):
    x, w, ids = inputs(32, 64, 64)
    bf = torch.bfloat16
    e = lambda *s, dtype=bf: torch.empty(*s, device="cuda", dtype=dtype)  # noqa: E731
    good = (ids, 2, e(32, 64))
    for mode, apart in (
        ("plain", good), ("silu", (ids[:31], 2, e(32, 64))), ("silu", (ids.long(), 2, e(32, 64))), ("silu", (ids, 2, e(32, 64, dtype=torch.float32))),
        ("silu", (ids, 2, e(31, 64))), ("silu", (ids, 2, e(32, 68)[:, :64])), ("silu", (ids, 2, e(64, 32).t())), ("silu", (ids.cpu(), 2, e(32, 64))),
    ):  # fmt: skip
        with pytest.raises((ValueError, TypeError, RuntimeError)):
            ops.gemm_tcgen05(x, w, e(32, 64) if mode == "plain" else e(32, 32), mode=mode, apart=apart)
    for gu, out, kw in (
        (e(32, 24, dtype=torch.float32), e(32, 12), {}), (e(32, 64), e(32, 32), dict(rows=(ids[:3], 2))), (e(32, 64), e(32, 32), dict(rows=(ids.long(), 2))),
        (e(32, 64, dtype=torch.float32), e(32, 32), dict(rows=(ids, 2))), (e(32, 24), e(32, 12), dict(rows=(ids, 2))), (e(32, 64), e(32, 32, dtype=torch.float32), {}),
        (e(1 + 32 * 64, dtype=torch.float32)[1:].view(32, 64), e(32, 32), {}),
    ):  # fmt: skip
        with pytest.raises((ValueError, TypeError, RuntimeError)):
            ops.silu_mul(gu, out, **kw)
