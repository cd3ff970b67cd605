"""Rotary positions and the per-head norms of queries and keys, against 64-bit numpy.

Tolerances.  An angle is reduced in 64 bits and rounded to 2^-25 of a turn
(1.9e-7 rad); sine and cosine add 2^-23 and the two products and their sum
2^-24 each, so a rotated element is within 6e-7 of its pair's amplitude: 1e-6 of
the row's largest element is allowed.  The norm sums 8 squares in a lane and
five shuffle steps, 13 * 2^-24 relative, halved by the root, and rsqrt is good to
2^-22: 1e-6 more.  A backward row adds a second such sum: 4e-6 of the row's
largest |g w| r.  A weight gradient sums n products whose parts carry 3e-6 each;
n additions in any order lose at most n 2^-24, here below 64 sequential ones in
a lane and 64 joins: 1e-5 of the sum of magnitudes.
"""

import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

SCALINGS = [None, {"type": "linear", "factor": 3.0}, {"type": "ntk", "factor": 4.0},
            {"type": "yarn", "factor": 8.0, "original_length": 512}]


def turned(x, rot, positions, back=False):
    """The rotation in 64 bits, the angles from the frequencies."""
    n = rot.dim // 2
    angle = np.asarray(positions, np.float64)[..., None, None] * rot.frequencies
    z = np.exp(1j * (-angle if back else angle)) * rot.factor
    y = x.astype(np.float64).copy()
    first, second = (slice(0, rot.dim, 2), slice(1, rot.dim, 2)) if rot.interleaved else \
        (slice(0, n), slice(n, rot.dim))
    w = (y[..., first] + 1j * y[..., second]) * z
    y[..., first], y[..., second] = w.real, w.imag
    return y


def close(got, want, rel, scale=None):
    got = got.numpy().astype(np.float64)
    size = np.abs(want).max(-1, keepdims=True) if scale is None else scale
    assert got.shape == want.shape
    assert np.all(np.abs(got - want) <= rel * size + 1e-30), float(np.max(np.abs(got - want) / (size + 1e-30)))


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("batch,seq,heads,dim,rot", [
    (1, 1, 1, 2, 2), (2, 3, 5, 64, 64), (3, 7, 2, 80, 20), (1, 130, 3, 128, 128), (2, 33, 1, 256, 256),
    (2, 5, 3, 31, 30), (1, 4, 2, 255, 16), (2, 9, 4, 96, 64), (1, 3, 2, 16, 8), (5, 1, 32, 128, 128)])
def test_rotation_and_its_gradient(interleaved, batch, seq, heads, dim, rot):
    import tynx_b200 as tx

    rng = np.random.default_rng(dim * 7 + seq)
    for k, scaling in enumerate(SCALINGS):
        rotary = tx.nn.Rotary(rot, interleaved=interleaved, scaling=scaling)
        x, dy = (rng.standard_normal((batch, seq, heads, dim)).astype(np.float32) for _ in range(2))
        per_batch = (rng.integers(-5, 100000, (batch, seq)), rng.integers(0, 2000, (seq,)), None)[k % 3]
        positions = np.arange(seq) if per_batch is None else per_batch
        positions = np.broadcast_to(positions, (batch, seq))
        X = tx.Tensor(x, requires_grad=True)
        Y = tx.nn.functional.rotary_embedding(X, rotary, None if per_batch is None else tx.Tensor(per_batch))
        Y.backward(tx.Tensor(dy))
        close(Y, turned(x, rotary, positions), 1e-6 * rotary.factor)
        close(X.grad, turned(dy, rotary, positions, back=True), 1e-6 * rotary.factor)
        if rot < dim:
            np.testing.assert_array_equal(Y.numpy()[..., rot:], x[..., rot:])


def test_far_positions_keep_their_angles():
    import tynx_b200 as tx

    rotary = tx.nn.Rotary(64)
    positions = np.array([0, 1, 2**20 + 1, 10**9 + 7, 2**40 + 3, -(2**33)])
    x = np.random.default_rng(0).standard_normal((1, 6, 2, 64)).astype(np.float32)
    # the reference reduces exactly: the frequencies' 64-bit values as rational numbers times the position
    from fractions import Fraction
    y = x.astype(np.float64).copy()
    for t, p in enumerate(positions):
        for i in range(32):
            f = Fraction(float(rotary._desc.turns[i])) * int(p)
            a = 2 * math.pi * float(f - round(f))
            lo, hi = x[0, t, :, i].astype(np.float64), x[0, t, :, i + 32].astype(np.float64)
            y[0, t, :, i], y[0, t, :, i + 32] = lo * math.cos(a) - hi * math.sin(a), lo * math.sin(a) + hi * math.cos(a)
    Y = tx.nn.functional.rotary_embedding(tx.Tensor(x), rotary, tx.Tensor(positions))
    # p * turns in 64 bits is good to 2^-53 p turns: 2^40 leaves 2^-13 of a turn at the first pair
    size = np.abs(x).max(-1, keepdims=True)
    bound = np.array([1e-6 + 2 * math.pi * abs(float(p)) * 2.0**-53 for p in positions])[None, :, None, None]
    assert np.all(np.abs(Y.numpy() - y) <= bound * 2 * size)


def norm_reference(x, w, rot, positions, eps, dy):
    x, w = x.astype(np.float64), w.astype(np.float64)
    r = 1.0 / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    y = turned(x * r * w, rot, positions)
    g = turned(dy, rot, positions, back=True)
    gw = g * w
    dx = r * (gw - x * r * (gw * x * r).mean(-1, keepdims=True))
    return y, dx, (g * x * r).sum((0, 1, 2)), np.abs(gw * r).max(-1, keepdims=True), np.abs(g * x * r).sum((0, 1, 2))


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("batch,seq,heads,kv,dim,rot", [
    (1, 1, 1, 1, 2, 2), (16, 1, 16, 4, 128, 128), (2, 65, 6, 3, 96, 64), (3, 7, 5, 1, 40, 20), (1, 300, 4, 4, 64, 64),
    (2, 11, 3, 1, 33, 32), (1, 9, 32, 8, 256, 256), (1, 5000, 2, 1, 16, 16)])
def test_norms_with_the_rotation(interleaved, batch, seq, heads, kv, dim, rot):
    import tynx_b200 as tx

    rng = np.random.default_rng(dim * 3 + seq)
    rotary = tx.nn.Rotary(rot, interleaved=interleaved, scaling=SCALINGS[(dim + seq) % 4])
    positions = rng.integers(0, 50000, (batch, seq))
    q, dq = (rng.standard_normal((batch, seq, heads, dim)).astype(np.float32) for _ in range(2))
    k, dk = (rng.standard_normal((batch, seq, kv, dim)).astype(np.float32) * 3 for _ in range(2))
    qw, kw = (1 + 0.2 * rng.standard_normal(dim).astype(np.float32) for _ in range(2))
    leaves = [tx.Tensor(a, requires_grad=True) for a in (q, k, qw, kw)]
    outs = tx.nn.functional.qk_norm_rotary(*leaves, rotary, tx.Tensor(positions), eps=1e-5)
    tx.backward(outs, [tx.Tensor(dq), tx.Tensor(dk)])
    for i, (x, w, dy) in enumerate(((q, qw, dq), (k, kw, dk))):
        y, dx, dw, size, total = norm_reference(x, w, rotary, positions, 1e-5, dy)
        close(outs[i], y, 2e-6 * rotary.factor)
        close(leaves[i].grad, dx, 4e-6, size)
        close(leaves[i + 2].grad, dw, 1e-5, total)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,rot", [(8, 8), (12, 12), (16, 8), (24, 10), (24, 24), (32, 32), (30, 16), (40, 20)])
def test_narrow_heads(interleaved, dim, rot):
    """Several rows share a warp."""
    import tynx_b200 as tx

    rng = np.random.default_rng(dim + rot)
    rotary = tx.nn.Rotary(rot, interleaved=interleaved)
    q, dq = (rng.standard_normal((3, 211, 7, dim)).astype(np.float32) for _ in range(2))
    k, dk = (rng.standard_normal((3, 211, 1, dim)).astype(np.float32) for _ in range(2))
    qw, kw = (1 + 0.2 * rng.standard_normal(dim).astype(np.float32) for _ in range(2))
    positions = np.broadcast_to(np.arange(211), (3, 211))
    leaves = [tx.Tensor(a, requires_grad=True) for a in (q, k, qw, kw)]
    outs = tx.nn.functional.qk_norm_rotary(*leaves, rotary, eps=1e-5)
    tx.backward(outs, [tx.Tensor(dq), tx.Tensor(dk)])
    for i, (x, w, dy) in enumerate(((q, qw, dq), (k, kw, dk))):
        y, dx, dw, size, total = norm_reference(x, w, rotary, positions, 1e-5, dy)
        close(outs[i], y, 2e-6)
        close(leaves[i].grad, dx, 4e-6, size)
        close(leaves[i + 2].grad, dw, 1e-5, total)
    x = tx.Tensor(q, requires_grad=True)
    y = tx.nn.functional.rotary_embedding(x, rotary)
    y.backward(tx.Tensor(dq))
    close(y, turned(q, rotary, positions), 1e-6)
    close(x.grad, turned(dq, rotary, positions, back=True), 1e-6)


def test_rows_of_zeros_and_repeated_calls():
    """A row of zeros has a finite norm through eps; the same inputs give the same bits."""
    import tynx_b200 as tx

    rotary = tx.nn.Rotary(64)
    rng = np.random.default_rng(1)
    q = rng.standard_normal((2, 400, 4, 64)).astype(np.float32)
    q[0, 3] = 0.0
    k = rng.standard_normal((2, 400, 2, 64)).astype(np.float32)
    w = np.ones(64, np.float32)
    results = []
    for _ in range(2):
        leaves = [tx.Tensor(a, requires_grad=True) for a in (q, k, w, w)]
        outs = tx.nn.functional.qk_norm_rotary(*leaves, rotary)
        tx.backward(outs, [tx.Tensor(q + 1), tx.Tensor(k)])
        results.append([t.numpy() for t in list(outs) + [x.grad for x in leaves]])
    assert all(np.isfinite(a).all() for a in results[0])
    np.testing.assert_array_equal(results[0][0][0, 3], 0.0)
    for a, b in zip(*results):
        np.testing.assert_array_equal(a, b)


def test_one_output_used_alone_and_empty_batches():
    import tynx_b200 as tx

    F, rotary = tx.nn.functional, tx.nn.Rotary(16)
    rng = np.random.default_rng(2)
    q, k = (rng.standard_normal((2, 5, 3, 16)).astype(np.float32) for _ in range(2))
    w = np.ones(16, np.float32)
    leaves = [tx.Tensor(a, requires_grad=True) for a in (q, k, w, w)]
    F.qk_norm_rotary(*leaves, rotary)[0].sum().backward()
    _, dx, dw, size, total = norm_reference(q, w, rotary, np.broadcast_to(np.arange(5), (2, 5)), 1e-6,
                                            np.ones_like(q))
    close(leaves[0].grad, dx, 4e-6, size)
    close(leaves[2].grad, dw, 1e-5, total)
    np.testing.assert_array_equal(leaves[1].grad.numpy(), 0.0)
    np.testing.assert_array_equal(leaves[3].grad.numpy(), 0.0)
    empty = tx.zeros(0, 5, 3, 16)
    assert F.rotary_embedding(empty, rotary).shape == (0, 5, 3, 16)
    leaves = [tx.zeros(2, 0, 3, 16).requires_grad_(), tx.zeros(2, 0, 1, 16).requires_grad_(),
              tx.Tensor(w, requires_grad=True), tx.Tensor(w, requires_grad=True)]
    outs = F.qk_norm_rotary(*leaves, rotary)
    tx.backward(outs, [tx.zeros(2, 0, 3, 16), tx.zeros(2, 0, 1, 16)])
    np.testing.assert_array_equal(leaves[2].grad.numpy(), 0.0)


def test_offsets_past_32_bits():
    import torch

    import tynx_b200 as tx

    rotary = tx.nn.Rotary(128)
    x = torch.ones(1, 600000, 32, 128, device="cuda")
    assert x.numel() > 2**31
    x[0, -1] = torch.arange(32 * 128, device="cuda").reshape(32, 128) / 4096.0
    y = torch.from_dlpack(tx.nn.functional.rotary_embedding(tx.from_dlpack(x), rotary))
    close(tx.from_dlpack(y[:, -2:].contiguous()), turned(x[:, -2:].cpu().numpy(), rotary, [[599998, 599999]]), 1e-6)


def test_unaligned_rows():
    """A view that starts off a 16-byte boundary takes the single-element path to the same values."""
    import torch

    import tynx_b200 as tx

    rotary = tx.nn.Rotary(64, interleaved=True)
    base = torch.randn(2 * 7 * 3 * 64 + 1, device="cuda")
    x = tx.from_dlpack(base[1:].reshape(2, 7, 3, 64))
    assert x.ptr % 16 == 4
    y = tx.nn.functional.rotary_embedding(x, rotary)
    close(y, turned(x.numpy(), rotary, np.broadcast_to(np.arange(7), (2, 7))), 1e-6)


def test_gradient_agrees_with_differences():
    import tynx_b200 as tx

    F, rotary = tx.nn.functional, tx.nn.Rotary(8, interleaved=True)
    rng = np.random.default_rng(3)
    arrays = [rng.standard_normal(s).astype(np.float32) for s in ((1, 3, 2, 8), (1, 3, 1, 8), (8,), (8,))]
    seeds = [rng.standard_normal(s).astype(np.float32) for s in ((1, 3, 2, 8), (1, 3, 1, 8))]

    def value(a):
        out = F.qk_norm_rotary(*[tx.Tensor(x) for x in a], rotary)
        return sum(float((o.numpy().astype(np.float64) * s).sum()) for o, s in zip(out, seeds))

    leaves = [tx.Tensor(a, requires_grad=True) for a in arrays]
    tx.backward(F.qk_norm_rotary(*leaves, rotary), [tx.Tensor(s) for s in seeds])
    for i, leaf in enumerate(leaves):
        way = rng.standard_normal(arrays[i].shape).astype(np.float32)
        h = 1e-2
        plus, minus = ([a + (h * s * way if j == i else 0) for j, a in enumerate(arrays)] for s in (1, -1))
        slope = (value(plus) - value(minus)) / (2 * h)
        want = float((leaf.grad.numpy().astype(np.float64) * way).sum())
        # third differences: h^2 / 6 times a third derivative of a few times the value's size
        assert abs(slope - want) <= 2e-3 * max(1.0, np.abs(leaf.grad.numpy() * way).sum())
