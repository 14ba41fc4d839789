"""Rotary frequencies where a stretched context's formula meets its ends (host arithmetic, no GPU)."""
import math

import pytest

from ltxattn import Failure, rotary_frequencies


def table(*args, **kw):
    f, magnitude = rotary_frequencies(*args, device="cpu", **kw)
    return f.tolist(), magnitude


@pytest.mark.parametrize("length", [1.0, 3.0, 6.25])
def test_yarn_stretches_every_pair_that_turns_less_than_slow(length):
    # in so few positions even the fastest pair turns less than once: all are divided by the factor
    plain, _ = table(8)
    got, _ = table(8, scaling="yarn", factor=2.0, trained_length=length)
    assert all(length * f / (2 * math.pi) < 1 for f in plain)
    assert got == [f / 2 for f in plain]


@pytest.mark.parametrize("length", [7.0, 64.0])
def test_yarn_keeps_the_fastest_pair_where_it_turns_at_least_once(length):
    # the ramp's ends are rounded outwards to whole pairs, so pair 0 is at its start
    plain, _ = table(8)
    got, _ = table(8, scaling="yarn", factor=2.0, trained_length=length)
    assert got[0] == plain[0] == 1.0 and got[-1] == plain[-1] / 2
