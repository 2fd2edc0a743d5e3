"""The scales of A and B in the workspace: powers of two, with which no value of theirs that the factors can make leaves FP16's range, and none much smaller
than that range allows. Held to the iteration on 20001 singular values from 0 to 1."""
import ctypes
import random

import numpy as np
import pytest

from oztt_amd import device as ozd
from oztt_amd import hip

S = np.linspace(0.0, 1.0, 20001)


def scales(a, b, c, steps):
    x, y = ctypes.c_double(), ctypes.c_double()
    hip().oz_rule_newton_schulz_scales(*map(ctypes.c_double, (a, b, c)), steps, ctypes.byref(x), ctypes.byref(y))
    return x.value, y.value


def largest(a, b, c, steps):
    """Of A and of B, over singular values from 0 to the largest that there are, as they stay below 8."""
    top = 1.0
    for _ in range(steps - 1):
        s = S * top
        top = min(max(top, float(np.abs(s * (a + b * s**2 + c * s**4)).max())), 8.0)
    q = (S * top) ** 2
    return float(q.max()), float(np.abs(b * q + c * q**2).max())


def check(a, b, c, steps):
    of_a, of_b = scales(a, b, c, steps)
    A, B = largest(a, b, c, steps)
    for scale, x in ((of_a, A), (of_b, B)):
        assert np.log2(scale) == int(np.log2(scale)) and 1.0 <= scale <= 16384.0
        assert scale == 1.0 or scale * x <= 32768.0 * 1.0001
    return of_a * A, of_b * B


def test_usual_factors():
    for steps in (1, 5, 100):
        A, B = check(*ozd.NEWTON_SCHULZ, steps)
        assert A > 16384.0 * 0.99 and B > 16384.0 * 0.5


@pytest.mark.parametrize("seed", range(40))
def test_other_factors(seed):
    rng = random.Random(seed)
    for _ in range(20):
        check(rng.uniform(-4, 8), rng.choice([0.0, rng.uniform(-12, 6)]), rng.choice([0.0, rng.uniform(-3, 9)]), rng.choice([1, 2, 3, 5, 12]))


def test_factors_of_nothing_and_of_much():
    assert scales(1.0, 0.0, 0.0, 5) == (16384.0, 16384.0)
    assert scales(1e30, -1e30, 1e30, 3) == (512.0, 1.0)
