"""The logarithm of a row's sum where many small exponentials lie beside a few large ones."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [1, 512, 1200])
@pytest.mark.parametrize("v", [70001, 128256])
def test_small_exponentials_are_not_lost_beside_large_ones(rows, v):
    """The first 4,096 logits of a row are 0, the rest -16.65: a thread that has summed sixteen ones loses sixteen of the rest
    (together just below half of 16's last place in 32 bits) every time it adds them, if it sums in 32 bits.

    Bounds: an exponential is off by 2^-21 of itself, a sum of sixteen of them by as much again (eight additions), the joined sums are
    in 64 bits; the score is rounded once, and the beam's own score puts it next to zero."""
    from kvforge_b200 import ops

    row = torch.full((v,), -16.65)
    row[:4096] = 0.0
    lse = float(torch.logsumexp(row.double(), 0))
    logits = row.cuda().repeat(rows, 1)
    scores = torch.full((rows,), lse, device="cuda")
    parents, tokens = (torch.full((rows, 2), -7, dtype=torch.int32, device="cuda") for _ in range(2))
    best = torch.full((rows, 2), 7.0, device="cuda")
    ops.beam_select(logits, scores, parents, tokens, best, ops.beam_workspace(rows, v, 2, "cuda"))
    want = scores.double()[:, None] - lse
    assert bool((parents == 0).all()) and tokens.tolist() == [[0, 1]] * rows
    off = float(((best.double() - want).abs() - want.abs() * 2.0**-24).max())
    assert off <= 2.0**-20
