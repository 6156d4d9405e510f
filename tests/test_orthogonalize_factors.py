"""Factors of ``navi_orthogonalize`` that its products' operands cannot hold are refused, without a GPU: addresses here
are never read (calls that are in order name no matrix)."""

from __future__ import annotations

import math
import random
import struct

import pytest

from navi_amd import _policy_native as native


def call(steps, factors):
    return native.lib().navi_orthogonalize(0, None, steps, *factors, 1e-6, None, None)


def largest(steps, factors, points=20001):
    """(singular values before a step, b s^2 + c s^4) at their largest, on a grid."""
    a, b, c = factors
    s, most, poly = 1.0, 1.0, 0.0
    for _ in range(steps):
        if s > 1e6:
            return math.inf, math.inf
        most = max(most, s)
        at = [s * i / (points - 1) for i in range(points)]
        poly = max(poly, max(abs(b * x ** 2 + c * x ** 4) for x in at))
        s = max(abs(a * x + b * x ** 3 + c * x ** 5) for x in at)
    return most, poly


FACTORS = [
    (5, (3.4445, -4.775, 2.0315)), (100, (3.4445, -4.775, 2.0315)), (100, (1.5, -0.5, 0.0)), (100, (1.875, -1.25, 0.375)),
    (1, (8.2872, -23.5959, 17.3004)), (1, (1e30, 0.0, 0.0)), (2, (7.8, 0.0, 0.0)), (2, (8.0, 0.0, 0.0)), (2, (-8.0, 0.0, 0.0)),
    (1, (0.0, 62.0, 0.0)), (1, (0.0, 64.0, 0.0)), (1, (0.0, 0.0, -62.0)), (1, (0.0, 0.0, 64.0)), (1, (0.0, 200.0, -200.0)),
    (1, (0.0, 300.0, -300.0)), (2, (20.0, -20.0, 0.0)), (2, (40.0, -40.0, 0.0)), (2, (30.0, -60.0, 30.0)), (2, (0.0, 0.0, 0.0)),
    (3, (2.0, 0.0, 0.0)), (4, (2.0, 0.0, 0.0)), (100, (1.01, 0.0, 0.0)), (100, (1.05, 0.0, 0.0)), (50, (3.0, 3.0, 3.0)),
    (2, (3e38, 3e38, 3e38)), (100, (-1.0, 2.0, -0.5)),
    (2, (22.0, -22.0, 1e-30)), (2, (22.0, -22.0, -1e-30)), (2, (10.0, -10.0, 1e-30)), (2, (22.0, -1e-30, -22.0)), (2, (-30.0, 1e-20, 30.0)),
]


@pytest.mark.parametrize("steps, factors", FACTORS, ids=str)
def test_factors_within_and_past_the_range(steps, factors):
    """65504 / 1024 = 63.97 is what float16 holds of A and P, 1.02 of which are left to roundings: 62.7, singular values
    of 7.92. (No factors here are within a part in a hundred of it.)"""
    s, poly = largest(steps, factors)
    room = 65504 / 1024 / 1.02
    assert min(abs(s * s / room - 1.0), abs(poly / room - 1.0)) > 0.01
    code = call(steps, factors)
    if max(s * s, poly) > room:
        assert code == native.NAVI_POLICY_E_ARG and "the factors take" in native.last_error()
    else:
        assert code == native.NAVI_POLICY_OK, native.last_error()


def test_factors_of_all_sizes():
    """Drawn ones against the grid, but for those within a part in 50 of the border."""
    rng, room, kinds = random.Random(7), 65504 / 1024 / 1.02, set()
    for _ in range(300):
        steps = rng.randint(1, 4)
        factors = tuple(rng.choice((-1, 1)) * 10 ** rng.uniform(-9, 1.9) if rng.random() < 0.9 else 0.0 for _ in range(3))
        factors = tuple(struct.unpack("f", struct.pack("f", x))[0] for x in factors)
        s, poly = largest(steps, factors, 2001)
        if min(abs(s * s / room - 1.0), abs(poly / room - 1.0)) < 0.02:
            continue
        past = max(s * s, poly) > room
        kinds.add(past)
        assert call(steps, factors) == (native.NAVI_POLICY_E_ARG if past else native.NAVI_POLICY_OK), (steps, factors)
    assert kinds == {False, True}


def test_what_is_no_number_is_refused():
    for factors in ((math.nan, 1.0, 1.0), (1.0, math.nan, 1.0), (1.0, 1.0, math.inf)):
        assert call(5, factors) == native.NAVI_POLICY_E_ARG
