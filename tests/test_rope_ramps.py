"""YaRN's ramp against its published form, where its ends lie beyond the pairs that there are (CPU)."""
import math

import pytest

from anvilq_b200 import ops


def published(R, theta, s, n, fast=32.0, slow=1.0):
    """Peng et al. 2023, as its authors' code has it: a pair's share of the interpolated frequency rises along
    the pairs' numbers, from that of `fast` turns in n tokens (rounded down, at least 0) to that of `slow`
    (rounded up, at most R - 1: there are R / 2 pairs)."""
    place = lambda turns: R * math.log(n / (turns * 2 * math.pi)) / (2 * math.log(theta))
    lo, hi = max(math.floor(place(fast)), 0), min(math.ceil(place(slow)), R - 1)
    hi = hi + 0.001 if hi == lo else hi
    out = []
    for i in range(R // 2):
        f, w = theta ** (-2.0 * i / R), min(1.0, max(0.0, (i - lo) / (hi - lo)))
        out.append(f / s * w + f * (1 - w))
    return out


@pytest.mark.parametrize("R,theta,s,n", [
    (16, 1e4, 8.0, 32768),        # the slowest pair turns 1.65 times in the original context
    (64, 1e4, 4.0, 131072), (64, 1e4, 4.0, 65536), (128, 1e4, 40.0, 1 << 20),
    (128, 1e6, 8.0, 32768), (64, 1e4, 8.0, 4096), (32, 500.0, 2.0, 8192), (2, 1e4, 2.0, 100),
    (64, 1e4, 16.0, 1 << 30),     # every pair turns more than 32 times
])
def test_the_ramp_ends_where_pairs_turn_slowly_enough(R, theta, s, n):
    inv, factor = ops.rope_frequencies(R, theta, dict(kind="yarn", factor=s, original=n), "cpu")
    for g, want in zip(inv.tolist(), published(R, theta, s, n)):
        assert math.isclose(g, want, rel_tol=1e-12)
    assert math.isclose(factor, 0.1 * math.log(s) + 1)


@pytest.mark.parametrize("R,theta,n", [(16, 1e4, 32768), (64, 1e4, 131072), (64, 1e4, 4), (16, 1e6, 6), (64, 1e4, 100),
                                       (64, 1e4, 1 << 40), (16, 1e4, 1 << 22)])
def test_only_slow_pairs_are_divided_and_only_fast_ones_stay(R, theta, n):
    """Below `slow` turns in the original context a pair is divided in full, above `fast` it stays; between, even
    the last pair is not divided in full unless the pair before the limit is."""
    s = 8.0
    inv, _ = ops.rope_frequencies(R, theta, dict(kind="yarn", factor=s, original=n), "cpu")
    for i, g in enumerate(inv.tolist()):
        f = theta ** (-2.0 * i / R)
        turns, step = n * f / (2 * math.pi), theta ** (2.0 / R)
        if turns < 1:
            assert math.isclose(g, f / s, rel_tol=1e-12)
        if turns > 32:
            assert g == f
        if turns / step > 1:             # the next pair, were there one, would turn more than once too
            assert g > f / s * (1 + 1e-6)
