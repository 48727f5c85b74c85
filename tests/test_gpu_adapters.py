"""Low-rank adapters of many requests at once against the formula in 64 bits."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from kvforge_b200 import ops as o

    return o


def make(ops, s, k, ends, rank, dtype, alternating=False, ranks=None, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + s * 3 + k)
    padded = -(-rank // 16) * 16
    a = torch.zeros(s, len(ends), padded, k, device="cuda")
    b = torch.zeros(s, ends[-1], padded, device="cuda")
    for i in range(s):
        r = rank if ranks is None else ranks[i]
        a[i, :, :r] = torch.randn(len(ends), r, k, generator=g, device="cuda") * k**-0.5
        b[i, :, :r] = torch.randn(ends[-1], r, generator=g, device="cuda")
    scales = 0.5 + torch.rand(s, generator=g, device="cuda")
    ranks = None if ranks is None else torch.tensor(ranks, dtype=torch.int32, device="cuda")
    return ops.AdapterBank(a.to(dtype), b.to(dtype), scales, ends, alternating, ranks)


def sections(bank):
    at = torch.arange(bank.n, device="cuda")
    if bank.alternating:
        return at // 8 % 2
    return torch.bucketize(at, torch.tensor(bank.ends, device="cuda"), right=True)


def formula(x, bank, ids, base):
    """(result, sums of absolute terms) in 64 bits."""
    out, mag = base.double().clone(), base.double().abs()
    sec = sections(bank)
    for s in sorted(set(ids)):
        if not 0 <= s < bank.size:
            continue
        rows = torch.tensor([i for i, t in enumerate(ids) if t == s], device="cuda")
        a, b, sc = bank.a[s].double(), bank.b[s].double(), float(bank.scales[s])
        xs = x[rows].double()
        for i in range(bank.sections):
            cols = torch.nonzero(sec == i)[:, 0]
            out[rows[:, None], cols] += (xs @ a[i].T * sc) @ b[cols].T
            mag[rows[:, None], cols] += (xs.abs() @ a[i].T.abs() * sc) @ b[cols].T.abs()
    return out, mag


def close(got, want, mag, dtype):
    """One rounding to the output's type, and sums in 32 bits: no sum is a chain of more than 64 roundings of partial sums (2^-18 of the
    absolute terms); where 16 bits come out, what is between the two products may be split in two 16-bit numbers (2^-17 of the terms more)."""
    half = torch.finfo(dtype).eps / 2
    assert torch.isfinite(got).all()
    bound = half * want.abs() + (2.0**-18 + (2.0**-17 if dtype == torch.bfloat16 else 0.0)) * mag
    assert ((got.double() - want).abs() <= bound).all(), float(((got.double() - want).abs() / bound).max())


def run(ops, x, bank, ids, base, in_place=False, err=None):
    t = torch.tensor(ids, dtype=torch.int32, device="cuda")
    groups = ops.AdapterGroups(max(1, len(ids)), bank.size, "cuda")
    ops.group_by_adapter(t, groups, err)
    if in_place:
        out = base.clone()
        ops.adapter_add(x, bank, groups, out)
    else:
        out = torch.full_like(base, float("nan"))
        ops.adapter_add(x, bank, groups, out, base=base)
    return out


def inputs(n, k, width, dtype, wide, seed=1):
    g = torch.Generator(device="cuda").manual_seed(seed + n)
    x = torch.randn(n, k, generator=g, device="cuda").to(dtype)
    base = torch.randn(n, width, generator=g, device="cuda")
    return x, base if wide else base.to(dtype)


def mixed_ids(n, s, seed=0):
    g = torch.Generator().manual_seed(seed + n)
    ids = torch.randint(-1, s, (n,), generator=g)
    at = n // 3
    ids[at : at + n // 2] = s - 1  # a portion of a prompt among the rest
    return ids.tolist()


CASES = [
    # adapters, K, ends, rank
    (1, 8, (8,), 16), (3, 64, (64, 96, 128), 8), (2, 72, (40, 48), 5), (5, 128, (128,), 1), (4, 200, (24, 32, 88, 96), 16), (3, 256, (520,), 33),
    (2, 2048, (2048, 2560, 3200), 16), (3, 4096, (1000,), 64), (2, 1000, (136, 400), 128), (2, 512, (256, 384, 512), 128), (1, 14336, (256,), 16), (70, 96, (80,), 12),
]  # fmt: skip


@pytest.mark.parametrize("dtype,wide", [(torch.bfloat16, False), (torch.bfloat16, True), (torch.float32, True)])
@pytest.mark.parametrize("s,k,ends,rank", CASES)
def test_adapter_add(ops, s, k, ends, rank, dtype, wide):
    bank = make(ops, s, k, ends, rank, dtype)
    for n in (1, 2, 7, 16, 17, 64, 150, 300):
        x, base = inputs(n, k, ends[-1], dtype, wide)
        ids = mixed_ids(n, s)
        want, mag = formula(x, bank, ids, base)
        close(run(ops, x, bank, ids, base), want, mag, base.dtype)
        close(run(ops, x, bank, ids, base, in_place=True), want, mag, base.dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("half", [8, 40, 104, 1024])
def test_adapter_add_alternating(ops, dtype, half):
    bank = make(ops, 3, 136, (half, 2 * half), 24, dtype, alternating=True)
    for n in (1, 5, 33, 260, 700):
        x, base = inputs(n, 136, 2 * half, dtype, False)
        ids = mixed_ids(n, 3)
        want, mag = formula(x, bank, ids, base)
        close(run(ops, x, bank, ids, base), want, mag, base.dtype)


@pytest.mark.parametrize("dtype,n", [(torch.bfloat16, 2048), (torch.bfloat16, 1999), (torch.bfloat16, 5000), (torch.float32, 1100)])
@pytest.mark.parametrize("kind", ["one", "own", "none", "portions", "scattered"])
def test_adapter_add_many_rows(ops, dtype, n, kind):
    s = 300 if kind == "own" else 6
    bank = make(ops, s, 264, (304, 352), 16, dtype)
    x, base = inputs(n, 264, 352, dtype, False)
    ids = {
        "one": [3] * n, "own": [i % s for i in range(n)], "none": [-1] * n, "portions": [(-1, 0, 5, 2)[i * 4 // n] for i in range(n)],
        "scattered": [(i * 7919) % 7 - 1 for i in range(n)],
    }[kind]  # fmt: skip
    want, mag = formula(x, bank, ids, base)
    close(run(ops, x, bank, ids, base), want, mag, base.dtype)
    if kind == "none":
        assert torch.equal(run(ops, x, bank, ids, base), base)


@pytest.mark.parametrize(
    "k,ends,rank,wide",
    [
        (64, (8, 16, 24), 16, False), (200, (136, 272, 408), 48, False), (264, (1000,), 128, False), (136, (520, 1032), 128, False), (136, (72, 80, 664), 112, False),
        (136, (520,), 64, True), (136, (136, 408), 32, True), (72, (264, 400), 64, True), (136, (3008,), 128, True),
    ],
)  # fmt: skip
def test_adapter_add_many_rows_of_every_shape(ops, k, ends, rank, wide):
    """Sections that end inside a piece, inner numbers that have room and that have none, ranks below the bank's, both results."""
    n = 901
    bank = make(ops, 4, k, ends, rank, torch.bfloat16, ranks=[rank, rank - 5, 0, 3])
    x, base = inputs(n, k, ends[-1], torch.bfloat16, wide)
    for ids in (mixed_ids(n, 4), [i * 4 // n for i in range(n)], [1] * 897 + [-1] * 4):
        want, mag = formula(x, bank, ids, base)
        for in_place in (False, True):
            close(run(ops, x, bank, ids, base, in_place), want, mag, base.dtype)


@pytest.mark.parametrize("half,n", [(8, 700), (136, 512), (136, 513), (136, 700), (1000, 2100)])
def test_adapter_add_many_rows_alternating(ops, half, n):
    bank = make(ops, 40, 136, (half, 2 * half), 24, torch.bfloat16, alternating=True)
    x, base = inputs(n, 136, 2 * half, torch.bfloat16, False)
    for ids in (mixed_ids(n, 40), [i % 40 for i in range(n)]):
        want, mag = formula(x, bank, ids, base)
        close(run(ops, x, bank, ids, base), want, mag, base.dtype)


def test_adapter_add_of_one_row_of_any_stride(ops):
    """How far it is to a row that there is not does not matter."""
    bank = make(ops, 2, 64, (64,), 16, torch.bfloat16)
    x, base = inputs(1, 64, 64, torch.bfloat16, False)
    want, mag = formula(x, bank, [1], base)
    one = lambda t: t.as_strided((1, 64), (3, 1))  # noqa: E731
    groups = ops.AdapterGroups(1, 2, "cuda")
    ops.group_by_adapter(torch.ones(1, dtype=torch.int32, device="cuda"), groups)
    out = torch.full_like(base, float("nan"))
    ops.adapter_add(one(x), bank, groups, one(out), base=one(base))
    close(out, want, mag, base.dtype)


def test_adapter_rows_without_an_adapter_stay_as_they_are(ops):
    bank = make(ops, 2, 64, (64,), 16, torch.bfloat16)
    for n in (3, 40, 600):
        x, base = inputs(n, 64, 64, torch.bfloat16, False)
        ids = [i % 3 - 1 for i in range(n)]
        x[::3] = float("nan")  # rows of padding may hold anything
        base[::3] = float("inf")
        for in_place in (False, True):
            out = run(ops, x, bank, ids, base, in_place)
            assert torch.equal(out[::3], base[::3]) and torch.isfinite(out[1::3]).all()


def test_adapter_ids_outside_the_bank(ops):
    bank = make(ops, 2, 64, (64,), 16, torch.bfloat16)
    for n in (4, 600):
        x, base = inputs(n, 64, 64, torch.bfloat16, False)
        err = torch.zeros(1, dtype=torch.int32, device="cuda")
        ids = [0, 2, -5, 1] + [-1] * (n - 4)
        out = run(ops, x, bank, ids, base, err=err)
        assert int(err) == 32
        want, mag = formula(x, bank, [0, -1, -1, 1] + [-1] * (n - 4), base)
        close(out, want, mag, base.dtype)


def test_adapter_ranks_below_the_banks(ops):
    ranks = [1, 0, 7, 16, 40, 64]
    for dtype in (torch.bfloat16, torch.float32):
        bank = make(ops, 6, 160, (96, 200), 64, dtype, ranks=ranks)
        for n in (6, 31, 500):
            x, base = inputs(n, 160, 200, dtype, False)
            ids = [i % 6 for i in range(n)]
            want, mag = formula(x, bank, ids, base)
            close(run(ops, x, bank, ids, base), want, mag, base.dtype)


def test_adapter_add_of_row_ranges(ops):
    """Column ranges of wider rows: x, base and result with strides of their own; what lies beside the result stays."""
    bank = make(ops, 2, 128, (72, 88), 16, torch.bfloat16)
    for n in (5, 400):
        g = torch.Generator(device="cuda").manual_seed(n)
        x = torch.randn(n, 400, generator=g, device="cuda").bfloat16()[:, 16:144]
        base = torch.randn(n, 104, generator=g, device="cuda").bfloat16()[:, 8:96]
        store = torch.full((n, 120), 5.0, device="cuda", dtype=torch.bfloat16)
        ids = mixed_ids(n, 2)
        groups = ops.AdapterGroups(1000, 2, "cuda")
        ops.group_by_adapter(torch.tensor(ids, dtype=torch.int32, device="cuda"), groups)
        ops.adapter_add(x, bank, groups, store[:, 16:104], base=base)
        want, mag = formula(x, bank, ids, base)
        close(store[:, 16:104], want, mag, torch.bfloat16)
        assert (store[:, :16] == 5).all() and (store[:, 104:] == 5).all()


def test_adapter_add_of_no_rows(ops):
    bank = make(ops, 2, 64, (64,), 16, torch.bfloat16)
    x, base = inputs(0, 64, 64, torch.bfloat16, False)
    assert run(ops, x, bank, [], base).shape == (0, 64)


def test_adapter_large_and_infinite_values(ops):
    """The numbers between the two products may be far beyond what 16 bits hold to a part in 2^17, and an infinity stays in its row."""
    bank = make(ops, 2, 64, (64,), 16, torch.bfloat16)
    for n in (4, 300):
        x, base = inputs(n, 64, 64, torch.bfloat16, True)
        x = (x.float() * 1e30).bfloat16()
        x[1, 5] = float("inf")
        ids = [i % 2 for i in range(n)]
        out = run(ops, x, bank, ids, base)
        keep = [i for i in range(n) if i != 1]
        want, mag = formula(x, bank, ids, base)
        close(out[keep], want[keep], mag[keep], torch.float32)
        assert not torch.isfinite(out[1]).any()


def test_adapter_groups_serve_many_banks_and_graphs(ops):
    """One grouping for all projections of a step, captured and replayed with other requests in place."""
    banks = [make(ops, 4, 64, (96,), 16, torch.bfloat16), make(ops, 4, 128, (64, 128), 32, torch.bfloat16)]
    for n in (8, 64, 512):
        ids = torch.full((n,), -1, dtype=torch.int32, device="cuda")
        groups = ops.AdapterGroups(n, 4, "cuda")
        xs = [inputs(n, b.k, b.n, torch.bfloat16, False, seed=i) for i, b in enumerate(banks)]
        outs = [torch.empty_like(base) for _, base in xs]

        def step():
            ops.group_by_adapter(ids, groups)
            for bank, (x, base), out in zip(banks, xs, outs):
                ops.adapter_add(x, bank, groups, out, base=base)

        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        for turn in range(3):
            chosen = mixed_ids(n, 4, seed=turn)
            ids.copy_(torch.tensor(chosen, dtype=torch.int32))
            graph.replay()
            for bank, (x, base), out in zip(banks, xs, outs):
                want, mag = formula(x, bank, chosen, base)
                close(out, want, mag, torch.bfloat16)


def test_adapter_add_on_another_stream_and_again(ops):
    bank = make(ops, 5, 512, (1024,), 16, torch.bfloat16)
    for n in (9, 700):
        x, base = inputs(n, 512, 1024, torch.bfloat16, False)
        ids = mixed_ids(n, 5)
        want = run(ops, x, bank, ids, base)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = run(ops, x, bank, ids, base)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(got, want)
        for _ in range(3):
            assert torch.equal(run(ops, x, bank, ids, base), want)


def test_adapter_bank_beyond_32_bits(ops):
    """A bank of more than 2^31 numbers: its last adapter."""
    s, k, n = 2400, 8192, 8192
    a = torch.zeros(s, 1, 128, k, dtype=torch.bfloat16, device="cuda")
    b = torch.zeros(s, n, 128, dtype=torch.bfloat16, device="cuda")
    a[s - 1] = torch.randn(1, 128, k, device="cuda") * k**-0.5
    b[s - 1] = torch.randn(n, 128, device="cuda")
    bank = ops.AdapterBank(a, b, torch.ones(s, device="cuda"))
    for rows in (3, 300):
        x, base = inputs(rows, k, n, torch.bfloat16, False)
        ids = [s - 1] * rows
        want, mag = formula(x, bank, ids, base)
        close(run(ops, x, bank, ids, base), want, mag, torch.bfloat16)
