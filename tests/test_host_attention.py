"""Rotary frequencies and the argument checks of the attention operators, without a GPU."""

import math
from types import SimpleNamespace

import numpy as np
import pytest

CTX = SimpleNamespace(index=0)


def t(*shape, dtype="float32", ctx=CTX):
    return SimpleNamespace(shape=tuple(shape), ndim=len(shape), dtype=dtype, ctx=ctx, device="cuda:0",
                           requires_grad=False)


def F():
    from tynx_b200.nn import functional

    return functional


def rotary(*a, **k):
    from tynx_b200.nn import Rotary

    return Rotary(*a, **k)


def test_frequencies():
    r = rotary(8)
    np.testing.assert_allclose(r.frequencies, [1.0, 0.1, 0.01, 0.001], rtol=1e-15)
    assert r.factor == 1.0 and not r.interleaved
    np.testing.assert_allclose([r._desc.turns[i] * 2 * math.pi for i in range(4)], r.frequencies, rtol=1e-15)
    np.testing.assert_allclose(rotary(8, scaling={"type": "linear", "factor": 4.0}).frequencies, r.frequencies / 4)
    ntk = rotary(8, scaling={"type": "ntk", "factor": 4.0}).frequencies
    np.testing.assert_allclose(ntk[[0, -1]], [1.0, 0.001 / 4], rtol=1e-12)
    assert rotary(2, scaling={"type": "ntk", "factor": 4.0}).frequencies[0] == 1.0


def test_blended_frequencies():
    plain = rotary(128)
    r = rotary(128, scaling={"type": "yarn", "factor": 8.0, "original_length": 4096})
    turns = 4096 * plain.frequencies / (2 * math.pi)
    np.testing.assert_allclose(r.frequencies[turns > 40], plain.frequencies[turns > 40])
    np.testing.assert_allclose(r.frequencies[turns < 0.8], plain.frequencies[turns < 0.8] / 8)
    ratio = r.frequencies / plain.frequencies
    assert np.all(np.diff(ratio) <= 0) and ratio[0] == 1.0 and abs(ratio[-1] - 0.125) < 1e-12
    assert abs(r.factor - (0.1 * math.log(8.0) + 1.0)) < 1e-15
    assert rotary(128, scaling={"type": "yarn", "factor": 8.0, "original_length": 4096,
                                "attention_factor": 1.0}).factor == 1.0


@pytest.mark.parametrize("args,kw,error", [
    ((7,), {}, ValueError), ((0,), {}, ValueError), ((258,), {}, ValueError), ((8.0,), {}, TypeError),
    ((8,), {"base": -1.0}, ValueError), ((8,), {"base": float("inf")}, ValueError),
    ((8,), {"scaling": {"type": "other", "factor": 2.0}}, ValueError),
    ((8,), {"scaling": {"type": "linear"}}, ValueError),
    ((8,), {"scaling": {"type": "linear", "factor": 0.5}}, ValueError),
    ((8,), {"scaling": {"type": "linear", "factor": float("nan")}}, ValueError),
    ((8,), {"scaling": {"type": "linear", "factor": 2.0, "original_length": 4}}, ValueError),
    ((8,), {"scaling": {"type": "yarn", "factor": 2.0}}, ValueError),
    ((8,), {"scaling": {"type": "yarn", "factor": 2.0, "original_length": 64, "beta_fast": 1.0}}, ValueError),
])
def test_rotary_refusals(args, kw, error):
    with pytest.raises(error):
        rotary(*args, **kw)


def test_rotary_embedding_refusals():
    r = rotary(8)
    f = F().rotary_embedding
    for x, rot, pos, error in [
            (t(2, 3, 4), r, None, ValueError), (t(2, 3, 4, 8, dtype="int64"), r, None, ValueError),
            (t(2, 3, 4, 6), r, None, ValueError), (t(2, 3, 4, 300), r, None, NotImplementedError),
            (t(2, 3, 4, 0), r, None, NotImplementedError),
            (t(2, 3, 4, 8), "r", None, TypeError), (t(2, 3, 4, 8), r, t(3), ValueError),
            (t(2, 3, 4, 8), r, t(4, dtype="int64"), ValueError), (t(2, 3, 4, 8), r, t(3, 2, dtype="int64"), ValueError),
            (t(2, 3, 4, 8), r, t(3, dtype="int64", ctx=SimpleNamespace(index=1)), ValueError)]:
        with pytest.raises(error):
            f(x, rot, pos)


def test_qk_norm_refusals():
    r = rotary(8)
    f = F().qk_norm_rotary
    q, k, w = t(2, 3, 4, 8), t(2, 3, 2, 8), t(8)
    for args, kw in [((t(3, 4, 8), k, w, w, r), {}), ((q, t(2, 4, 2, 8), w, w, r), {}),
                     ((q, t(2, 3, 2, 6), w, w, r), {}), ((q, k, t(6), w, r), {}),
                     ((q, k, w, t(8, dtype="int64"), r), {}), ((q, k, w, w, r), {"eps": -1.0}),
                     ((q, k, w, w, r), {"eps": float("nan")}), ((q, k, w, w, r, t(2)), {}),
                     ((q, t(2, 3, 2, 8, ctx=SimpleNamespace(index=1)), w, w, r), {})]:
        with pytest.raises(ValueError):
            f(*args, **kw)


def test_differential_attention_refusals():
    f = F().differential_attention
    q, k, v, lam = t(2, 3, 8, 16), t(2, 5, 4, 16), t(2, 5, 2, 32), t(4)
    n = t(2, dtype="int64")
    other = SimpleNamespace(index=1)
    for args, kw, error in [
            ((t(2, 3, 8), k, v, lam), {}, ValueError),
            ((t(2, 3, 7, 16), k, v, lam), {}, ValueError),          # half a pair of maps
            ((t(2, 3, 6, 16), k, v, t(3)), {}, ValueError),          # 3 heads over 2 key heads
            ((q, t(2, 5, 3, 16), v, lam), {}, ValueError),
            ((q, t(2, 5, 0, 16), v, lam), {}, ValueError),
            ((q, t(1, 5, 4, 16), v, lam), {}, ValueError),
            ((q, t(2, 5, 4, 8), v, lam), {}, ValueError),
            ((q, k, t(2, 4, 2, 32), lam), {}, ValueError),
            ((q, k, t(2, 5, 4, 32), lam), {}, ValueError),
            ((q, k, v, t(8)), {}, ValueError),
            ((q, k, v, t(4, dtype="int64")), {}, ValueError),
            ((q, k, v, t(4, ctx=other)), {}, ValueError),
            ((q, k, v, lam), {"key_lengths": t(2)}, ValueError),
            ((q, k, v, lam), {"key_lengths": t(3, dtype="int64")}, ValueError),
            ((q, k, v, lam), {"key_lengths": t(2, dtype="int64", ctx=other)}, ValueError),
            ((q, k, v, lam), {"scale": float("inf")}, ValueError),
            ((t(2, 3, 8, 65), t(2, 5, 4, 65), v, lam), {}, NotImplementedError),
            ((q, k, t(2, 5, 2, 129), lam), {}, NotImplementedError),
            ((q, k, v, lam), {"key_lengths": n, "scale": float("nan")}, ValueError)]:
        with pytest.raises(error):
            f(*args, **kw)


def test_backward_refusals():
    from tynx_b200 import backward

    y = t(2, 3)
    y.requires_grad = True
    for tensors, grads in [([y], []), ([t(2, 3)], [t(2, 3)]), ([y], [t(3, 2)]), ([y], [t(2, 3, dtype="int64")])]:
        with pytest.raises(ValueError):
            backward(tensors, grads)


def test_values_that_do_not_fit_the_call_are_refused():
    from tynx_b200 import backward

    args = t(2, 3, 8, 16), t(2, 5, 4, 16), t(2, 5, 2, 32), t(4)
    for start in (1 << 64, -(1 << 31)):
        with pytest.raises(ValueError, match="query_start"):
            F().differential_attention(*args, causal=True, query_start=start)
    y = t(2, 3)
    y.requires_grad = True
    with pytest.raises(ValueError, match="gradient on"):
        backward([y], [t(2, 3, ctx=SimpleNamespace(index=1))])
