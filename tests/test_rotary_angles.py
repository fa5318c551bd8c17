"""CPU: the angle that a RotaryPlan's integers give at a position, against the formula in 60
decimal digits.  Off by |position| 2^-65 turns for the fraction's rounding and |position| f e
for the frequency, a double, with e
  2^-52  for the power alone (within one unit in its last place);
  2^-51  with the quotient or the blend of a scaling, up to two roundings of 2^-53;
  2^-50  with ntk's base, five roundings of 2^-53 taken to a power below 1;
  2^-49  where 2 i / dim is rounded itself, by 2^-53 of an exponent whose logarithm is below
         ln(theta) < 14 (ntk's base < 16)."""

from __future__ import annotations

import math
from decimal import Decimal, getcontext

import pytest

from treemoe_spec_amd.kernels.rotary import RotaryPlan

PI = Decimal("3.14159265358979323846264338327950288419716939937510582097494459230781640629")


def _frequency(i, dim, theta, scaling):
    """Turns a position of pair i."""
    theta, s = Decimal(theta), Decimal(scaling["factor"]) if scaling else Decimal(1)
    kind = scaling["type"] if scaling else None
    if kind == "ntk":
        theta *= s ** (Decimal(dim) / (dim - 2))
    f = theta ** (Decimal(-2 * i) / dim) / (2 * PI)
    if kind == "linear":
        return f / s
    if kind == "yarn":
        span = scaling["original_max_position"] / (2 * math.pi)
        edge = lambda turns: dim * math.log(span / turns) / (2 * math.log(float(theta)))  # noqa: E731
        lo, hi = max(math.floor(edge(32)), 0), min(math.ceil(edge(1)), dim - 1)
        ramp = min(max(Decimal(i - lo) / max(hi - lo, 1), Decimal(0)), Decimal(1))
        return f * (1 - ramp) + f / s * ramp
    return f


@pytest.mark.parametrize("dim,theta", [(128, 10 ** 6), (64, 10 ** 4), (16, 500000),
                                       (80, 10 ** 6), (112, 10 ** 4)])
@pytest.mark.parametrize("scaling", [None, {"type": "linear", "factor": 3},
                                     {"type": "ntk", "factor": 4},
                                     {"type": "yarn", "factor": 8, "original_max_position": 4096}])
def test_angles(dim, theta, scaling):
    getcontext().prec = 60
    plan = RotaryPlan(dim, float(theta), scaling=scaling, device="cpu")
    steps = 52 if scaling is None else 50 if scaling["type"] == "ntk" else 51
    if dim & (dim - 1):
        steps = 49
    for i, u in enumerate(plan.turns.tolist()):
        f = _frequency(i, dim, theta, scaling)
        for pos in (1, 4097, 2 ** 20, 2 ** 30 + 7, 2 ** 40 + 12345, -77777):
            got = Decimal(pos * u % 2 ** 64) / 2 ** 64
            off = abs(got - pos * f) % 1
            off = min(off, 1 - off)
            bound = abs(pos) * (Decimal(2) ** -65 + f * Decimal(2) ** -steps)
            assert off <= bound, (i, pos, off, bound)
