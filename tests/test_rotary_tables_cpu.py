"""Frequencies of stretched rotary ranges against their definition, pair by pair in plain Python."""
import math

import pytest
import torch

from apla_amd import rotary as R


def yarn_pair(i, rot, base, factor, trained, fast=32.0, slow=1.0):
    """Pair i by the published method: the pair index at which a full range makes `turns` turns is rot ln(trained / (2 pi turns)) / (2 ln base); the
    ramp runs between the two indices, rounded outwards and cut to 0 .. rot - 1."""
    at = lambda turns: rot * math.log(trained / (2 * math.pi * turns)) / (2 * math.log(base))      # noqa: E731
    lo, hi = max(math.floor(at(fast)), 0), min(math.ceil(at(slow)), rot - 1)
    r = 1.0 if i >= hi else min(max((i - lo) / (hi - lo), 0.0), 1.0)
    f = base ** (-2 * i / rot)
    return f * (1 - r) + f / factor * r


@pytest.mark.parametrize("rot,base,trained", [(64, 1e4, 4096), (64, 1e4, 131072), (64, 100.0, 1370), (32, 100.0, 1370), (16, 1e4, 1 << 20), (64, 5e5, 8192), (64, 100.0, 1 << 20), (64, 1e4, 100), (64, 1e4, 5)])
@pytest.mark.parametrize("factor", [1.0, 4.0, 40.0])
def test_yarn_frequencies(rot, base, trained, factor):
    got = R.rotary_frequencies(rot, base, scaling="yarn", factor=factor, trained=trained)
    want = torch.tensor([yarn_pair(i, rot, base, factor, trained) for i in range(rot // 2)], dtype=torch.float64)
    assert bool(((got - want).abs() <= 1e-12 * want).all())


def test_yarn_last_pair_of_a_long_trained_range_is_divided_in_part():
    """The last of 32 pairs turns 2.78 times over 131072 positions at base 1e4, more than beta_slow = 1: the ramp runs from 22 to 35, (31 - 22) / 13 of
    the way there divides by 4 a share of 9 / 13."""
    f, y = R.rotary_frequencies(64), R.rotary_frequencies(64, scaling="yarn", factor=4.0, trained=131072)
    assert abs(float(y[31] / f[31]) - (4 / 13 + 9 / 13 / 4)) < 1e-12
