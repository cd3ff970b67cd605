"""The rotary frequencies against 60-digit arithmetic.

With u = 2^-53 and w = base^(-2 i / dim): the exponent's rounding, u of itself, changes the power by ln(1 / w) u;
the power is good to an ulp (2 u), 2 pi to u / 2, the division by it to u: ln(1 / w) + 3.5 in all.  Dividing by a
linear factor adds 1.  The stretched base of ntk is off by its exponent's rounding times the logarithm of its
factor, at most 2 ln f for dim >= 4, an ulp of its power and the product's rounding, 2 ln f + 3.
"""

import math
from decimal import Decimal, localcontext

import pytest

TWO_PI = 2 * Decimal("3.14159265358979323846264338327950288419716939937510582097494459")


def exact(base, dim, i, scaling):
    """Turns a position, in the caller's precision."""
    b, f = Decimal(base), Decimal((scaling or {}).get("factor", 1.0))
    if scaling and scaling["type"] == "ntk":
        b = b * (f.ln() * dim / (dim - 2)).exp()
    w = (b.ln() * (-2 * i) / dim).exp()
    return (w / f if scaling and scaling["type"] == "linear" else w) / TWO_PI


@pytest.mark.parametrize("scaling", [None, {"type": "linear", "factor": 3.0}, {"type": "ntk", "factor": 8.0}],
                         ids=["plain", "linear", "ntk"])
@pytest.mark.parametrize("base,dim", [(1e4, 64), (1e4, 96), (1e6, 80), (5e5, 128), (1e7, 142), (100.0, 202), (1e4, 4)])
def test_turns(base, dim, scaling):
    from tynx_b200.nn import Rotary

    rotary = Rotary(dim, base=base, scaling=scaling)
    more = {None: 0.0, "linear": 1.0, "ntk": 3.0 + 2 * math.log(8.0)}[scaling and scaling["type"]]
    with localcontext() as context:
        context.prec = 60
        for i in range(dim // 2):
            want = exact(base, dim, i, scaling)
            off = abs(Decimal(rotary._desc.turns[i]) / want - 1) * 2**53
            assert off <= Decimal(3.5 + more - math.log(float(want * TWO_PI))), (i, off)
