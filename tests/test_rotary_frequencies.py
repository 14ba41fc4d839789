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


@pytest.mark.parametrize("kw", [
    dict(scaling="ntk", theta=1e308, factor=8.0),      # the grown base is infinite: all pairs but the first would stand still
    dict(scaling="linear", factor=1e-320),             # the first pair's angle is infinite
    dict(theta=1e-320, rotary_dim=256, scaling="linear", factor=1e-5),
])
def test_frequencies_that_leave_the_range_are_refused(kw):
    with pytest.raises(Failure) as e:
        rotary_frequencies(**{"rotary_dim": 64, "device": "cpu", **kw})
    assert e.value.kind == "arg"


@pytest.mark.parametrize("rotary_dim", [2 ** 32 + 64, 2 ** 31, -2 ** 32 + 2, 2 ** 70])
def test_sizes_that_are_no_32_bit_numbers_are_refused(rotary_dim):
    # as an int32 the first is 64, the third 2; the answer must not be a table of that size
    with pytest.raises(Failure) as e:
        rotary_frequencies(rotary_dim, device="cpu")
    assert e.value.kind == "shape"


def test_a_rotary_dim_that_is_no_whole_number_is_refused():
    for bad in (64.5, "64", None):
        with pytest.raises((Failure, TypeError)):
            rotary_frequencies(bad, device="cpu")
