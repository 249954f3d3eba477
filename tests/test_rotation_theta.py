"""Frequencies above one radian a position: right to the last bit of their table as far as they are taken."""
from decimal import Decimal, localcontext

import pytest

from qutai_b200.rotary import Rotation

PI = Decimal("3.14159265358979323846264338327950288419716939937510582097494")


@pytest.mark.parametrize("theta", [1e-15, 1e-3, 0.5, 1.0, 1e30])
def test_fractions_of_a_turn(theta):
    with localcontext() as context:
        context.prec = 90
        for i, turns in enumerate(Rotation(8, theta=theta)._turns):
            want = Decimal(theta) ** (Decimal(-2 * i) / 8) / (2 * PI) % 1 * 2 ** 64
            assert abs(want - turns) <= 1 or abs(want - turns) >= 2 ** 64 - 1


@pytest.mark.parametrize("theta", [1e-16, 1e-25, 1e-300, -1.0])
def test_other_thetas_are_refused(theta):
    with pytest.raises(ValueError):
        Rotation(8, theta=theta)
