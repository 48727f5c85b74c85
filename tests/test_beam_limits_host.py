"""Length penalties that the floats cannot carry are refused before a search begins."""

from __future__ import annotations

import math

import pytest

from kvforge_b200 import BeamParams
from kvforge_b200.engine.beam import BeamGroup, _Beam
from kvforge_b200.engine.scheduler import RequestRejectedError


@pytest.mark.parametrize("penalty", [64.0, -64.0, 61.5, -57.0, 1.0, 0.6, 0.0, -2.0])
@pytest.mark.parametrize("limit", [1, 4096, 65535, 65536, 131072, 2**31])
def test_every_length_that_is_allowed_has_a_score(penalty, limit):
    """Scores are finite and not zero (a sum of log probabilities lies between the least float above zero and 104 a token, the
    logarithm of that float) from the first token to the last that is allowed."""
    try:
        group = BeamGroup([1], BeamParams(length_penalty=penalty), set(), limit)
    except RequestRejectedError:
        assert abs(penalty) * math.log2(limit) > 800  # nothing else is refused
        return
    for length in {1, 2, limit // 2 + 1, limit}:
        for logprob in (-(2.0**-149), -1.0, -104.0 * length):
            score = group.score(logprob, length)
            assert math.isfinite(score) and score < 0.0


def test_a_search_does_not_end_in_an_overflow():
    """The step at which a hypothesis reaches a length whose power is none."""
    for penalty in (64.0, -64.0):
        with pytest.raises(RequestRejectedError, match="length_penalty"):
            group = BeamGroup([1], BeamParams(num_beams=1, length_penalty=penalty), {9}, 140000)
            group.beams = [_Beam("a", [5] * 131071, -3.0)]
            group.choose([0], [9], [-4.0])
