"""The fractions of a turn in a rotation plan against 60-digit arithmetic. No device.

The fraction is cut to 64 bits (2^-64). f / 2 pi itself is a long double: five roundings of it (power, its scale, the constant,
the division; powl counts as two halves) and that of the exponent, which moves the power by its logarithm, each 2^-64 of it."""
import math
import os
from decimal import Decimal, getcontext

import pytest

import __graft_entry__ as ge

PI = Decimal("3.14159265358979323846264338327950288419716939937510582097494")


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(os.path.join(ge.PKG_DIR, "libiris_b200.so")):
        ge.build()
    return ge.load_package().load()


@pytest.mark.parametrize("dims,scales,theta,one", [
    ((32, 32, 32, 32), None, 2000.0, False), ((32, 48, 48), (24.0, 0.625, -1.0), 256.0, False), ((128,), (1.0,), 1e6, True),
    ((16, 56, 56), (1000.0, -3.5, 1.0), 10000.0, True), ((2, 126), None, 0.01, False)])
def test_fractions_are_as_exact_as_the_kernels_say(lib, dims, scales, theta, one):
    getcontext().prec = 60
    plan = lib.rope_axes(dims, scales, theta, one, 128)
    j = 0
    for a, dim in enumerate(dims):
        for i in range(dim // 2):
            power = Decimal(2 * j) / 128 if one else Decimal(2 * i) / dim
            turns = Decimal(scales[a] if scales else 1.0) * (-power * Decimal(theta).ln()).exp() / (2 * PI)
            off = abs(Decimal(plan.turn[j]) / 2 ** 64 - turns % 1) % 1
            off = float(min(off, 1 - off))
            assert off <= 2.0 ** -64 * (1 + abs(float(turns)) * (5 + float(power) * abs(math.log(theta)))), (a, i)
            j += 1
