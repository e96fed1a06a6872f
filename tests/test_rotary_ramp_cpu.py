"""Ramps of rotary frequencies against the rule by turns, not against the plan's own arithmetic."""
import math

import pytest
import torch

from shift_b200.ops import packed

# theta, rotated columns, original context, factor
SETTINGS = [(1.0e4, 128, 131072, 4.0), (1.0e4, 16, 32768, 4.0), (1.0e4, 128, 4096, 16.0), (5.0e5, 128, 131072, 8.0),
            (1.0e6, 96, 4096, 16.0), (1.0e4, 64, 1 << 20, 2.0), (100.0, 32, 65536, 8.0), (1.0e4, 64, 3, 8.0), (1.0e4, 2, 4096, 4.0),
            (1.0e4, 64, 64, 8.0)]


@pytest.mark.parametrize("theta,rot,original,factor", SETTINGS)
@pytest.mark.parametrize("fast,slow", [(32.0, 1.0), (16.0, 2.0), (64.0, 0.5)])
def test_pairs_go_by_how_often_they_turn(theta, rot, original, factor, fast, slow):
    plan = packed.Rotary(rot, theta, scaling=packed.RotaryScaling("ramp", factor, original, fast, slow), device="cpu")
    last = 0.0
    for i, f in enumerate(plan.freq.tolist()):
        plain = math.exp(-2.0 * i / rot * math.log(theta))
        turns = original * plain / (2 * math.pi)
        share = (1 - f / plain) / (1 - 1 / factor)         # 0: as it was, 1: divided
        assert -1e-9 <= share <= 1 + 1e-9 and share >= last - 1e-9
        last = share
        if turns > fast * (1 + 1e-9):
            assert abs(share) < 1e-9, (i, turns)
        if turns < slow * (1 - 1e-9):
            assert abs(share - 1) < 1e-9, (i, turns)
        if turns > slow * (1 + 1e-9):
            assert share < 1 - 1e-9, (i, turns)            # not all the way


@pytest.mark.parametrize("theta,rot,original,factor", SETTINGS[:7])
def test_ramp_of_the_published_rule(theta, rot, original, factor):
    """Linear between the pairs (real numbers, then floor and ceiling) that turn 32 times and once, held to [0, columns - 1]."""
    def pair_of(turns):
        return rot * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(theta))

    low, high = max(math.floor(pair_of(32)), 0), min(math.ceil(pair_of(1)), rot - 1)
    i = torch.arange(rot // 2, dtype=torch.float64)
    keep = 1 - ((i - low) / ((high - low) if high != low else 0.001)).clamp(0, 1)
    plain = theta ** (-2 * i / rot)
    want = plain / factor * (1 - keep) + plain * keep
    plan = packed.Rotary(rot, theta, scaling=packed.RotaryScaling("ramp", factor, original), device="cpu")
    assert torch.allclose(plan.freq, want, rtol=1e-12)


@pytest.mark.parametrize("factor,magnitude", [(0.25, 1.0), (1.0, 1.0), (1e-8, 1.0), (8.0, 0.1 * math.log(8) + 1)])
def test_contexts_no_longer_than_the_original_keep_their_magnitude(factor, magnitude):
    plan = packed.Rotary(64, 1.0e4, scaling=packed.RotaryScaling("ramp", factor, 4096), device="cpu")
    assert plan.magnitude == magnitude
