"""The choice of beams and the copies that follow it, each alone against a plain form in 64 bits."""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from kvforge_b200 import ops as o

    return o


# ------------------------------------------------------------------ the choice


def plain_select(logits, scores, prompts, k):
    """(parents, tokens, best, the smallest distance between neighbours in order) on the CPU in 64 bits."""
    x, s = logits.double().cpu(), scores.double().cpu()
    v = x.shape[1]
    beams = x.shape[0] // prompts
    every = s[:, None] + (x - torch.logsumexp(x, dim=1, keepdim=True))
    bad = torch.isnan(x).any(1) | (x == math.inf).any(1) | ~torch.isfinite(s) | (x == -math.inf).all(1)
    every[bad] = -math.inf
    every = every.view(prompts, beams * v)
    parents, tokens, best, gap = [], [], [], math.inf
    for row in every:
        order = torch.sort(-row, stable=True).indices[: k + 1]
        val = row[order]
        fin = val[torch.isfinite(val)]
        d = fin[:-1] - fin[1:]
        d = d[d > 0]
        if len(d):
            gap = min(gap, float(d.min()))
        order, val = order[:k], val[:k]
        pad = k - len(order)
        none = val == -math.inf
        parents.append(torch.where(none, -1, order // v).tolist() + [-1] * pad)
        tokens.append(torch.where(none, -1, order % v).tolist() + [-1] * pad)
        best.append(val.tolist() + [-math.inf] * pad)
    return parents, tokens, torch.tensor(best, dtype=torch.float64), gap


def select(ops, logits, scores, prompts, k, workspace=None):
    rows, v = logits.shape
    ws = workspace if workspace is not None else ops.beam_workspace(rows, v, k, "cuda")
    parents, tokens = (torch.full((prompts, k), -7, dtype=torch.int32, device="cuda") for _ in range(2))
    best = torch.full((prompts, k), 7.0, device="cuda")
    ops.beam_select(logits, scores, parents, tokens, best, ws)
    return parents, tokens, best


def check(ops, logits, scores, prompts, k, ordered=True, workspace=None):
    parents, tokens, best = select(ops, logits, scores, prompts, k, workspace)
    p, t, b, gap = plain_select(logits, scores, prompts, k)
    # a score is rounded to 32 bits once; the logarithm of the sum is off by less than 2e-7: an exponential by at most 2^-21
    # of itself (its argument is a rounded difference of at most 2^5 where it weighs anything, its function two units in the last place)
    same = best.cpu().double()
    assert torch.equal(torch.isfinite(same), torch.isfinite(b))
    fin = torch.isfinite(b)
    assert ((same - b)[fin].abs() <= b[fin].abs() * 2.0**-24 + 2.0**-20).all()
    if ordered:
        assert gap > 2.0**-20, "the case's scores lie too close to one another to ask for an order"
        assert parents.tolist() == p
        assert tokens.tolist() == t


@pytest.mark.parametrize(
    "prompts,beams,v,k",
    [
        (1, 1, 1, 1), (1, 1, 5, 3), (1, 4, 7, 8), (2, 2, 31, 4), (3, 5, 257, 10), (1, 4, 1000, 64), (2, 64, 300, 64), (1, 64, 1, 64),
        (5, 3, 4099, 6), (1, 8, 32003, 16), (2, 4, 128256, 8), (1, 1, 128257, 2), (40, 8, 8191, 16), (130, 4, 2049, 8), (700, 1, 513, 1),
    ],
)  # fmt: skip
def test_beam_select_random(ops, prompts, beams, v, k):
    g = torch.Generator().manual_seed(prompts * 7 + beams * 11 + v * 13 + k)
    logits = 3 * torch.randn(prompts * beams, v, generator=g)
    scores = -10 * torch.rand(prompts * beams, generator=g)
    gap = plain_select(logits, scores, prompts, k)[3]
    check(ops, logits.cuda(), scores.cuda(), prompts, k, ordered=gap > 2.0**-20)


@pytest.mark.parametrize("shape", ["rising", "falling", "constant", "zeros", "steps", "spike", "tiny", "last"])
@pytest.mark.parametrize("v", [100, 5000, 70001])
def test_beam_select_hard_rows(ops, shape, v):
    """Orders and ties that a search which counts on chance would not get through: rows in order, rows of one value, few values."""
    k, beams = 16, 4
    at = torch.arange(v, dtype=torch.float32)
    row = {
        "rising": at * 0.01, "falling": -at * 0.01, "constant": torch.full((v,), -3.25), "zeros": torch.where(at % 2 == 0, 0.0, -0.0), "steps": (at % 7) * 0.5,
        "spike": torch.where(at == v // 2, 80.0, 0.0), "tiny": torch.where(at % 3 == 0, 1e-42, -1e-42), "last": torch.where(at >= v - 20, at - v, -50.0 + 0 * at),
    }[shape]  # fmt: skip
    logits = row.repeat(beams, 1).cuda()
    equal = torch.full((beams,), -1.5, device="cuda")
    parents, tokens, best = select(ops, logits, equal, 1, k)
    # all beams have the same scores: the k best are the row's best logits, of each the beams in turn (equal scores: lowest beam first, then token)
    every = row.double() - torch.logsumexp(row.double(), 0) - 1.5
    if shape == "tiny":  # logits whose difference is lost beside the logarithm: only values are held
        assert ((best.cpu().double() - every.max()).abs() < 2.0**-20).all()
        return
    flat = every.repeat(beams)
    order = torch.sort(-flat, stable=True).indices[:k]
    assert (best[0].cpu().double() - flat[order]).abs().max() <= 2.0**-18
    assert parents[0].tolist() == (order // v).tolist()
    assert tokens[0].tolist() == (order % v).tolist()


def test_beam_select_masks_and_dead_beams(ops):
    g = torch.Generator().manual_seed(3)
    beams, v, k = 6, 3001, 12
    logits = torch.randn(4 * beams, v, generator=g)
    scores = -torch.rand(4 * beams, generator=g)
    logits[torch.rand(logits.shape, generator=g) < 0.3] = -math.inf
    scores[1:beams] = -math.inf  # the first choice of a prompt: one beam is alive
    logits[beams + 1] = -math.inf  # nothing left
    logits[beams + 2, 17] = math.nan
    logits[beams + 3, 3000] = math.inf
    scores[beams + 4] = math.nan
    logits[2 * beams : 3 * beams] = -math.inf  # a prompt with three candidates in all
    logits[2 * beams + 2, 5] = 1.0
    logits[2 * beams + 5, 2999] = -4.0
    logits[2 * beams + 5, 0] = -3.0
    logits[3 * beams :] = -math.inf  # and one without any
    logits[3 * beams, :] = torch.finfo(torch.float32).min  # the lowest value of the type is a value
    check(ops, logits.cuda(), scores.cuda(), 4, k)
    scores[3 * beams] = math.inf
    parents, tokens, best = select(ops, logits.cuda(), scores.cuda(), 4, k)
    assert parents[3].tolist() == [-1] * k and tokens[3].tolist() == [-1] * k and (best[3] == -math.inf).all()


def test_beam_select_more_places_than_candidates(ops):
    logits = torch.tensor([[0.5, -1.0, 2.0], [0.25, 3.0, -2.0]])
    check(ops, logits.cuda(), torch.tensor([-1.0, -2.0]).cuda(), 1, 16)


@pytest.mark.parametrize("offset,stride", [(0, 1000), (1, 1003), (3, 1024), (2, 2001)])
def test_beam_select_rows_off_alignment(ops, offset, stride):
    g = torch.Generator().manual_seed(5)
    v, rows = 999, 6
    store = torch.full((offset + rows * stride + 8,), 1e9, device="cuda")  # what lies between the rows must not be read as logits
    logits = store[offset:].as_strided((rows, v), (stride, 1))
    logits.copy_(torch.randn(rows, v, generator=g))
    check(ops, logits, -torch.rand(rows, generator=g).cuda(), 2, 6)


def test_beam_select_workspace_serves_smaller_calls_and_graphs(ops):
    g = torch.Generator().manual_seed(9)
    ws = ops.beam_workspace(32, 20000, 16, "cuda")
    cases = []
    for prompts, beams, v, k in ((4, 8, 20000, 16), (1, 3, 77, 5), (8, 4, 9999, 8), (2, 2, 20000, 1), (4, 8, 20000, 16)):
        logits, scores = torch.randn(prompts * beams, v, generator=g).cuda(), -torch.rand(prompts * beams, generator=g).cuda()
        check(ops, logits, scores, prompts, k, ordered=False, workspace=ws)
        cases.append((logits, scores, prompts, k))
    # two captured calls share the workspace, replayed in turn with new numbers in place
    graphs = []
    for logits, scores, prompts, k in cases[:3]:
        outs = [torch.empty((prompts, k), dtype=d, device="cuda") for d in (torch.int32, torch.int32, torch.float32)]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ops.beam_select(logits, scores, *outs, ws)
        graphs.append((graph, outs))
    for turn in range(3):
        for (graph, outs), (logits, scores, prompts, k) in zip(graphs, cases):
            logits.copy_(torch.randn(logits.shape, generator=g))
            graph.replay()
            want = select(ops, logits, scores, prompts, k)
            assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_beam_select_on_another_stream(ops):
    g = torch.Generator().manual_seed(2)
    logits, scores = torch.randn(12, 30000, generator=g).cuda(), -torch.rand(12, generator=g).cuda()
    want = select(ops, logits, scores, 3, 8)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = select(ops, logits, scores, 3, 8)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_beam_select_is_the_same_every_time(ops):
    g = torch.Generator().manual_seed(4)
    logits, scores = torch.randn(64, 128256, generator=g).cuda(), -torch.rand(64, generator=g).cuda()
    first = select(ops, logits, scores, 8, 16)
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(select(ops, logits, scores, 8, 16), first))
    # and a prompt's choice does not depend on its neighbours
    alone = select(ops, logits[8:16], scores[8:16], 1, 16)
    assert torch.equal(alone[0][0], first[0][1]) and torch.equal(alone[1][0], first[1][1])


# ------------------------------------------------------------------ the copies


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("entries,blocks,heads,bs,d,dv", [(1, 4, 1, 1, 8, 8), (3, 9, 2, 16, 16, 48), (2, 12, 3, 4, 3, 5), (4, 9, 1, 16, 576, 0), (16, 40, 8, 16, 64, 64), (2, 9, 5, 32, 2, 6)])
def test_copy_pages(ops, dtype, entries, blocks, heads, bs, d, dv):
    g = torch.Generator().manual_seed(blocks * d)
    k = torch.randn(entries, blocks, heads, bs, d, generator=g).to(dtype).cuda()
    v = torch.randn(entries, blocks, heads, bs, dv, generator=g).to(dtype).cuda() if dv else None
    order = torch.randperm(blocks, generator=g).tolist()
    n = max(1, blocks // 3)
    dst, src = order[:n], [order[n], *[order[n + i % (blocks - n)] for i in range(n - 1)]]
    for tokens in (None, [(7 * i) % (bs + 1) for i in range(n)], [bs + 3] * n):
        want = [t.clone() if t is not None else None for t in (k, v)]
        for t in want:
            if t is not None:
                for i in range(n):
                    m = bs if tokens is None else min(tokens[i], bs)
                    t[:, dst[i], :, :m] = t[:, src[i], :, :m]
        got = [t.clone() if t is not None else None for t in (k, v)]
        ops.copy_pages(got[0], got[1], i32(src), i32(dst), None if tokens is None else i32(tokens))
        assert torch.equal(got[0], want[0]) and (v is None or torch.equal(got[1], want[1]))


def test_copy_pages_outside_the_pool_copies_nothing(ops):
    k = torch.randn(2, 6, 2, 4, 8, device="cuda")
    v = torch.randn(2, 6, 2, 4, 8, device="cuda")
    want_k, want_v = k.clone(), v.clone()
    want_k[:, 5], want_v[:, 5] = k[:, 0], v[:, 0]
    ops.copy_pages(k, v, i32([-1, 6, 2, 3, 0, 1, 4]), i32([2, 3, -1, 6, 5, 1, 2**31 - 1]))
    assert torch.equal(k, want_k) and torch.equal(v, want_v)
    ops.copy_pages(k, v, i32([]), i32([]))
    ops.copy_pages(k, v, i32([0, 1]), i32([2, 3]), i32([0, -4]))
    assert torch.equal(k, want_k) and torch.equal(v, want_v)


def test_copy_pages_beyond_32_bits(ops):
    """A cache of more than 2^32 bytes: the last pages of its last layer."""
    k = torch.zeros(3, 40000, 8, 16, 128, dtype=torch.bfloat16, device="cuda")
    k[2, 39990] = 3.0
    ops.copy_pages(k, None, i32([39990, 39990]), i32([39999, 1]), i32([16, 5]))
    assert (k[2, 39999] == 3.0).all() and (k[2, 1, :, :5] == 3.0).all() and (k[2, 1, :, 5:] == 0).all()
    assert float(k.sum(dtype=torch.float64)) == 3.0 * 8 * 128 * (16 + 16 + 5)


@pytest.mark.parametrize("widths", [[4], [1], [512, 512], [5280, 4096, 7], [262144, 280576, 149504], [4097] * 20])
@pytest.mark.parametrize("slots", [2, 9])
def test_copy_states(ops, widths, slots):
    states = [torch.randn(slots, w, device="cuda") for w in widths]
    states.append(torch.randn(slots, 2, 3, 4, device="cuda"))
    src, dst = ([0], [1]) if slots == 2 else ([4, 4, 0, 8], [1, 2, 7, 3])
    want = [t.clone() for t in states]
    for t in want:
        t[dst] = t[src]
    ops.copy_states(ops.StateTable(states), i32([*src, -1, slots]), i32([*dst, 0, 0]))
    assert all(torch.equal(a, b) for a, b in zip(states, want))


def test_copy_states_of_column_ranges(ops):
    """Slots that are wider than the state (a column range of a wider tensor) keep what lies beside it."""
    wide = torch.randn(6, 40, device="cuda")
    want = wide.clone()
    want[2, 3:30], want[5, 3:30] = wide[0, 3:30], wide[1, 3:30]
    ops.copy_states(ops.StateTable([wide[:, 3:30]]), i32([0, 1]), i32([2, 5]))
    assert torch.equal(wide, want)


def test_copies_replay_in_a_graph(ops):
    k = torch.randn(3, 8, 2, 16, 32, device="cuda")
    state = torch.randn(8, 1000, device="cuda")
    table = ops.StateTable([state])
    src, dst, tokens = i32([0, 0]), i32([1, 2]), i32([16, 3])
    graph = torch.cuda.CUDAGraph()
    keep = k.clone(), state.clone()
    ops.copy_pages(k, None, src, dst, tokens)
    ops.copy_states(table, src, dst)
    with torch.cuda.graph(graph):
        ops.copy_pages(k, None, src, dst, tokens)
        ops.copy_states(table, src, dst)
    k.copy_(keep[0])
    state.copy_(keep[1])
    src.copy_(i32([5, 6]))
    dst.copy_(i32([7, 0]))
    graph.replay()
    want = keep[0].clone(), keep[1].clone()
    want[0][:, 7], want[0][:, 0, :, :3] = want[0][:, 5], want[0][:, 6, :, :3]
    want[1][7], want[1][0] = want[1][5], want[1][6]
    assert torch.equal(k, want[0]) and torch.equal(state, want[1])
