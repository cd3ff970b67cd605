"""Angles of far positions, from frequencies of 60 digits.

An angle p w is off by (5 + ln(1 / w)) 2^-53 of itself at most, one 2^-53 more where the position itself passes 2^53
and is rounded; a rotated element is off by that of its pair's amplitude, and by 1e-6 as near positions are.
"""

import math
from decimal import Decimal, localcontext

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("base,dim", [(1e4, 96), (1e6, 80)])
def test_far_positions(base, dim, interleaved):
    import tynx_b200 as tx
    from tests.test_host_rotary_frequencies import TWO_PI, exact

    rotary = tx.nn.Rotary(dim, base=base, interleaved=interleaved)
    positions = [1, 2**22 + 1, 10**9 + 7, 2**40 + 3, -(2**33) - 1, 2**50 + 1, 2**53 - 1, 2**61 + 1, -(2**63)]
    x = np.random.default_rng(dim).standard_normal((1, len(positions), 2, dim)).astype(np.float32)
    y = tx.nn.functional.rotary_embedding(tx.Tensor(x), rotary, tx.Tensor(np.array(positions, np.int64))).numpy()
    with localcontext() as context:
        context.prec = 60
        for i in range(dim // 2):
            a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + dim // 2)
            turns = exact(base, dim, i, None)
            for t, p in enumerate(positions):
                turn = turns * p
                angle = 2 * math.pi * float(turn - turn.to_integral_value())
                off = float(abs(turn) * TWO_PI) * (5 + (abs(p) > 2**53) - math.log(float(turns * TWO_PI))) * 2.0**-53
                lo, hi = x[0, t, :, a].astype(np.float64), x[0, t, :, b].astype(np.float64)
                bound = (off + 1e-6) * np.hypot(lo, hi)
                c, s = math.cos(angle), math.sin(angle)
                assert np.all(np.abs(y[0, t, :, a] - (lo * c - hi * s)) <= bound), (i, p)
                assert np.all(np.abs(y[0, t, :, b] - (lo * s + hi * c)) <= bound), (i, p)
