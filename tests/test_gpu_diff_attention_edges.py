"""Differential attention: the precision of its products, calls without gaps, memory off 16-byte boundaries and
caches with room to spare, against 64-bit numpy.

Precision.  An operand is a pair of fp16 within 2^-22 of its value, and the product of two tails, 2^-22 of the
product, is left out.  As independent errors of a uniform distribution the two operands' add up to
sqrt(2) 2^-22 / sqrt(3) = 1.9e-7 of a sum's norm; the tensor core adds a tile's large products with truncation, at
most 8 times half an ulp of 2^-23 on average, 4.8e-7.  One stage of products: 5.2e-7.  An output has two stages, a
gradient four (scores, dP, D and its own product): 2.1e-6 where all add up.  Pairs of bf16, 2^-17 an operand after
the rounding of both parts, would be at 32 times the first part, 6e-6 a stage.
"""

import gc

import numpy as np
import pytest

from tests.test_gpu_diff_attention import arrays, call, check, reference

pytestmark = pytest.mark.gpu

STAGE = 5.2e-7


@pytest.mark.parametrize("case", [
    (1, 128, 128, 2, 2, 64, 128, True, 0),
    (2, 300, 513, 4, 2, 64, 64, False, 0),
    (1, 1024, 1024, 2, 1, 64, 128, True, 0),
    (25, 62, 62, 6, 2, 64, 72, True, 0),      # a group's heads in one tile
    (2, 4, 700, 4, 2, 64, 128, True, 696),    # few queries
    (4, 64, 2048, 4, 2, 64, 128, True, 1984),
], ids=lambda c: "x".join(map(str, c[:7])))
def test_precision_of_fp16_pairs(case):
    B, T, S, H, Hk, d, dv, causal, start = case
    q, k, v, lam, dout = arrays(B, T, S, H, Hk, d, dv, T + S + 5)
    val, _ = reference(q, k, v, lam, dout, d ** -0.5, causal, start, None)
    got = call(q, k, v, lam, dout, causal=causal, query_start=start, lengths=None)
    for name, g, w in zip(("out", "dq", "dk", "dv", "dlam"), got, val):
        stages = 2 if name == "out" else 4
        off = np.linalg.norm(g.numpy() - w) / np.linalg.norm(w)
        assert off <= stages * STAGE, (name, off)


CLOSE = [
    (8, 1, 700, 4, 2, 64, 128),      # few queries, joined
    (2, 40, 2000, 4, 2, 64, 128),    # ranges of keys, joined
    (40, 50, 50, 4, 2, 64, 128),     # a group's heads in one tile
    (2, 300, 300, 6, 1, 40, 72),     # key blocks of single heads, summed
]


@pytest.mark.parametrize("shape", CLOSE, ids=lambda c: "x".join(map(str, c)))
def test_calls_without_gradients_and_without_gaps(shape):
    """Every call of a burst has the bits of one that ran alone."""
    import tynx_b200 as tx

    F = tx.nn.functional
    sets = [[tx.Tensor(x) for x in arrays(*shape, 60 + i)[:4]] for i in range(3)]
    with tx.no_grad():
        alone = []
        for s in sets:
            tx.synchronize()
            out = F.differential_attention(*s, causal=True)
            tx.synchronize()
            alone.append(out.numpy())
        burst = [F.differential_attention(*sets[i % 3], causal=True) for i in range(48)]
    for i, out in enumerate(burst):
        np.testing.assert_array_equal(out.numpy(), alone[i % 3])


@pytest.mark.parametrize("shape", CLOSE, ids=lambda c: "x".join(map(str, c)))
def test_training_calls_without_gaps(shape):
    """The same forward and backward, with nothing uploaded between the calls."""
    import tynx_b200 as tx

    F = tx.nn.functional
    data = [arrays(*shape, 70 + i) for i in range(3)]
    alone = []
    for a in data:
        tx.synchronize()
        got = call(*a, causal=True, lengths=None)
        tx.synchronize()
        alone.append([t.numpy() for t in got])
    leaves = [[tx.Tensor(x, requires_grad=True) for x in data[i % 3][:4]] for i in range(18)]
    douts = [tx.Tensor(a[4]) for a in data]
    tx.synchronize()
    outs = []
    for i, s in enumerate(leaves):
        out = F.differential_attention(*s, causal=True)
        out.backward(douts[i % 3])
        outs.append(out)
    for i, s in enumerate(leaves):
        for g, w in zip([outs[i]] + [t.grad for t in s], alone[i % 3]):
            np.testing.assert_array_equal(g.numpy(), w)


@pytest.mark.parametrize("off", [1, 2, 3])
@pytest.mark.parametrize("case", [
    (2, 1, 300, 4, 2, 64, 128), (3, 7, 130, 2, 1, 32, 64), (1, 130, 200, 2, 2, 64, 128), (50, 43, 43, 3, 1, 64, 64),
    (2, 150, 70, 3, 1, 40, 72)], ids=lambda c: "x".join(map(str, c)))
def test_memory_off_16_byte_boundaries(case, off):
    """q, k, v and the output's gradient start 4, 8 or 12 bytes behind a boundary."""
    import torch

    import tynx_b200 as tx

    B, T, S, H, Hk, d, dv = case
    q, k, v, lam, dout = arrays(*case, 80 + off)
    lengths = [S - 3 * (b % 2) for b in range(B)]

    def shifted(a):
        base = torch.empty(a.size + off, device="cuda")
        base[off:] = torch.from_numpy(a).reshape(-1).cuda()
        t = tx.from_dlpack(base[off:].reshape(a.shape))
        assert t.ptr % 16 == 4 * off
        return t

    val, tol = reference(q, k, v, lam, dout, d ** -0.5, True, S - T, lengths)
    leaves = [shifted(a).requires_grad_() for a in (q, k, v, lam)]
    n = tx.Tensor(np.array(lengths))
    out = tx.nn.functional.differential_attention(*leaves, causal=True, key_lengths=n)
    out.backward(shifted(dout))
    check([out.detach()] + [t.grad for t in leaves], val, tol)
    with tx.no_grad():
        check([tx.nn.functional.differential_attention(*leaves, causal=True, key_lengths=n)], val[:1], tol[:1])


@pytest.mark.parametrize("queries", [1, 5, 40])
def test_a_cache_with_room_to_spare(queries):
    """Lengths far below the keys' memory: the values are those of the filled part, the rest is not read."""
    import tynx_b200 as tx

    B, S, H, Hk, d, dv, full = 5, 32768, 4, 2, 16, 32, 3000
    q, k, v, lam, dout = arrays(B, queries, full, H, Hk, d, dv, 90 + queries)
    lengths = [full, 1, 0, 777, 128]
    val, tol = reference(q, k, v, lam, dout, d ** -0.5, False, 0, lengths)
    cache_k, cache_v = np.full((B, S, 2 * Hk, d), np.nan, np.float32), np.full((B, S, Hk, dv), np.inf, np.float32)
    for b, n in enumerate(lengths):
        cache_k[b, :n], cache_v[b, :n] = k[b, :n], v[b, :n]
    got = call(q, cache_k, cache_v, lam, dout, causal=False, query_start=0, lengths=lengths)
    for i in (2, 3):
        g = got[i].numpy()
        for b, n in enumerate(lengths):
            np.testing.assert_array_equal(g[b, n:], 0.0)
        got[i] = tx.Tensor(g[:, :full])
    check(got, val, tol)
    with tx.no_grad():
        out = tx.nn.functional.differential_attention(
            *(tx.Tensor(a) for a in (q, cache_k, cache_v, lam)), key_lengths=tx.Tensor(np.array(lengths)))
    check([out], val[:1], tol[:1])
    gc.collect()
