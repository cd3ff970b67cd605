"""Differential attention against 64-bit numpy.

Tolerances.  A product's operands carry at least 16 bits (a bf16 head and
tail): each is within 2^-18 of its value and the product of the two tails is
left out, 3 * 2^-18 of |a b| a product in all, E below.  So with c_ij = scale
sum |q k| a score is within E c_ij, a weight within 2 E max_j c_ij of itself
(numerator and sum), and an output within sum_j (a1 + |lam| a2) |v| times that
and E for its own product.  The gradients' bounds follow the same way through
dP (E sum |dO| |v|), D (the outputs' bound), dS and the last product.  Sums in
fp32 add less than a tenth of this.  What is held in 16 bits has a floor besides:
an fp16 head and tail are each rounded to half of 2^-24, 2^-24 in all, and a
weight carries at least 2^8 (2^13 / (1 + |lam|) in the backward), so it is within
2^-32 (1 + |lam|) however small it is; a score gradient, scaled so that 2 max|dO|
max|v| lies in [2^12, 2^14), is within 2^-24 / 2^12 of that bound.  Those bounds are for the worst case at
every element; over a whole tensor errors of this kind are independent, about
1e-6 of its norm, and 1e-5 is allowed.
"""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

E = 3 * 2.0**-18


def reference(q, k, v, lam, dout, scale, causal, start, lengths):
    """Values and elementwise error bounds of (out, dq, dk, dv, dlam)."""
    B, T, H2, d = q.shape
    S, Hk = k.shape[1], k.shape[2] // 2
    H, dv = H2 // 2, v.shape[3]
    q, k, v, lam, dout = (a.astype(np.float64) for a in (q, k, v, lam, dout))
    val = [np.zeros((B, T, H, dv)), np.zeros_like(q), np.zeros_like(k), np.zeros_like(v), np.zeros(H)]
    tol = [np.zeros_like(a) for a in val]
    i, j = np.arange(T)[:, None], np.arange(S)[None, :]
    for b in range(B):
        n = S if lengths is None else int(lengths[b])
        ok = (j < n) & ((j <= i + start) if causal else True)
        ok = np.broadcast_to(ok, (T, S))[:, :n]
        if n == 0:
            continue
        for h in range(H):
            kv = h // (H // Hk)
            vv, g = v[b, :n, kv], dout[b, :, h]
            a, ea = [], []
            for m in range(2):
                qm, km = q[b, :, 2 * h + m], k[b, :n, 2 * kv + m]
                s = np.where(ok, qm @ km.T * scale, -np.inf)
                top = s.max(-1, keepdims=True)
                p = np.where(ok, np.exp(s - np.where(np.isfinite(top), top, 0.0)), 0.0)
                a.append(p / np.maximum(p.sum(-1, keepdims=True), 1e-300))
                c = np.abs(qm) @ np.abs(km).T * abs(scale)
                ea.append(2 * E * np.where(ok, c, 0.0).max(-1, keepdims=True) + 4e-7)  # relative error of the weights
            floor = 2.0**-32 * (1 + abs(lam[h])) * ok
            w = a[0] - lam[h] * a[1]
            ew = floor + a[0] * ea[0] + abs(lam[h]) * a[1] * ea[1]
            wabs = a[0] + abs(lam[h]) * a[1]
            val[0][b, :, h] = w @ vv
            tol[0][b, :, h] = (ew + E * wabs) @ np.abs(vv)
            dp = g @ vv.T
            edp = E * np.abs(g) @ np.abs(vv).T
            val[3][b, :n, kv] += w.T @ g
            tol[3][b, :n, kv] += (ew + E * wabs).T @ np.abs(g)
            for m in range(2):
                f = scale if m == 0 else -lam[h] * scale
                D = (a[m] * dp).sum(-1, keepdims=True)
                eD = ((a[m] * (ea[m] + E)) @ np.abs(vv) * np.abs(g)).sum(-1, keepdims=True)
                ds = a[m] * (dp - D) * f
                bound = 2 * np.linalg.norm(dout[b, :, h], axis=-1).max() * np.linalg.norm(vv, axis=-1).max()
                eds = abs(f) * 2.0**-36 * bound * ok + abs(f) * a[m] * (edp + eD + (ea[m] + 4e-7) * np.abs(dp - D))
                val[1][b, :, 2 * h + m] = ds @ k[b, :n, 2 * kv + m]
                tol[1][b, :, 2 * h + m] = (eds + E * np.abs(ds)) @ np.abs(k[b, :n, 2 * kv + m])
                val[2][b, :n, 2 * kv + m] += ds.T @ q[b, :, 2 * h + m]
                tol[2][b, :n, 2 * kv + m] += (eds + E * np.abs(ds)).T @ np.abs(q[b, :, 2 * h + m])
                if m == 1:
                    val[4][h] -= D.sum()
                    tol[4][h] += eD.sum() + 1e-5 * np.abs(D).sum()
    return val, tol


def check(got, val, tol):
    for name, g, w, t in zip(("out", "dq", "dk", "dv", "dlam"), got, val, tol):
        g = g.numpy().astype(np.float64)
        assert g.shape == w.shape and np.isfinite(g).all(), name
        off = np.abs(g - w)
        assert np.all(off <= 1.1 * t + 1e-30), (name, float((off / (t + 1e-30)).max()))
        norm = np.linalg.norm(w)
        if norm > 1e-3:
            assert np.linalg.norm(g - w) <= 1e-5 * norm, (name, np.linalg.norm(g - w) / norm)


def call(q, k, v, lam, dout, **kw):
    import tynx_b200 as tx

    leaves = [tx.Tensor(a, requires_grad=True) for a in (q, k, v, lam)]
    lengths = kw.pop("lengths")
    out = tx.nn.functional.differential_attention(
        *leaves, key_lengths=None if lengths is None else tx.Tensor(np.asarray(lengths, np.int64)), **kw)
    out.backward(tx.Tensor(dout))
    return [out.detach()] + [t.grad for t in leaves]


def arrays(B, T, S, H, Hk, d, dv, seed):
    rng = np.random.default_rng(seed)
    n = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
    return n(B, T, 2 * H, d), n(B, S, 2 * Hk, d), n(B, S, Hk, dv), rng.random(H).astype(np.float32), n(B, T, H, dv)


CASES = [
    # B, T, S, H, Hk, d, dv, causal, start, lengths
    (1, 1, 1, 1, 1, 1, 1, False, 0, None),
    (2, 1, 7, 2, 1, 8, 16, False, 0, None),
    (2, 5, 5, 3, 3, 40, 72, True, 0, None),
    (1, 64, 64, 2, 2, 64, 128, False, 0, None),
    (1, 128, 128, 1, 1, 64, 128, True, 0, None),
    (2, 129, 129, 2, 1, 64, 128, True, 0, [129, 65]),
    (3, 33, 200, 4, 2, 32, 64, True, 167, [200, 0, 1]),
    (2, 200, 31, 2, 2, 64, 64, True, -169, None),   # the first rows see nothing
    (1, 70, 300, 6, 2, 63, 127, False, 0, [257]),
    (4, 100, 100, 3, 1, 64, 128, True, 0, [0, 1, 63, 100]),
    (1, 300, 513, 2, 2, 16, 32, True, 40, None),
    (2, 3, 130, 8, 2, 64, 128, True, 127, [130, 64]),
    (1, 257, 640, 1, 1, 64, 100, False, 0, None),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "x".join(map(str, c[:7])))
def test_values_and_gradients(case):
    B, T, S, H, Hk, d, dv, causal, start, lengths = case
    q, k, v, lam, dout = arrays(B, T, S, H, Hk, d, dv, T + S)
    val, tol = reference(q, k, v, lam, dout, d ** -0.5, causal, start, lengths)
    check(call(q, k, v, lam, dout, causal=causal, query_start=start, lengths=lengths), val, tol)


@pytest.mark.parametrize("queries", [1, 3])
@pytest.mark.parametrize("keys", [1, 63, 64, 65, 1000, 5000])
def test_few_queries_against_many_keys(queries, keys):
    import tynx_b200 as tx

    q, k, v, lam, dout = arrays(3, queries, keys, 4, 2, 64, 128, keys)
    lengths = [keys, max(0, keys - 7), keys // 2]
    val, tol = reference(q, k, v, lam, dout, 0.125, False, 0, lengths)
    with tx.no_grad():
        out = tx.nn.functional.differential_attention(*(tx.Tensor(a) for a in (q, k, v, lam)),
                                                      key_lengths=tx.Tensor(np.array(lengths)))
    check([out], val[:1], tol[:1])


@pytest.mark.parametrize("case", [
    (2, 64, 200, 4, 2, 64, 128, True, 136, None),
    (1, 43, 43, 3, 1, 64, 128, True, 0, None),              # 129 rows: the last token's heads in two tiles
    (3, 5, 333, 32, 1, 16, 33, True, 328, [333, 0, 7]),
    (1, 129, 129, 4, 2, 40, 64, True, -1, [128]),           # the first query sees nothing
    (2, 64, 4100, 4, 2, 64, 128, False, 0, [4100, 515]),    # keys in ranges, some of them empty
    (1, 20, 1500, 6, 2, 64, 72, True, 1480, None),
    (1, 300, 300, 10, 2, 64, 64, True, 0, None),
], ids=lambda c: "x".join(map(str, c[:7])))
def test_heads_that_share_keys_without_a_gradient(case):
    """Queries of a group's heads share tiles where nothing is kept for a backward."""
    import tynx_b200 as tx

    B, T, S, H, Hk, d, dv, causal, start, lengths = case
    q, k, v, lam, dout = arrays(B, T, S, H, Hk, d, dv, T + S + 1)
    val, tol = reference(q, k, v, lam, dout, d ** -0.5, causal, start, lengths)
    with tx.no_grad():
        out = tx.nn.functional.differential_attention(
            *(tx.Tensor(a) for a in (q, k, v, lam)), causal=causal, query_start=start,
            key_lengths=None if lengths is None else tx.Tensor(np.asarray(lengths, np.int64)))
    check([out], val[:1], tol[:1])


@pytest.mark.parametrize("weight", [1.0, -40.0, 0.0])
@pytest.mark.parametrize("case", [
    (25, 62, 62, 6, 2, 64, 72, True, 0, [62, 5, 0, 1, 61] * 5),
    (13, 26, 285, 12, 4, 64, 64, False, 0, None),
    (3, 64, 300, 64, 2, 16, 24, True, 236, [299, 300, 1]),  # 32 heads a group: 2048 rows
    (5, 7, 50, 33, 1, 8, 16, False, 0, None),
    (26, 50, 20, 6, 2, 40, 128, True, -30, None),           # the first queries see nothing
    (75, 64, 64, 2, 1, 64, 128, True, 0, None),             # exactly one tile
    (50, 43, 43, 3, 1, 64, 128, True, 0, None),             # 129 rows
    (30, 2, 9, 6, 2, 33, 65, True, 7, None),
    (2, 62, 62, 6, 2, 64, 72, True, 0, [62, 5]),            # too few heads: a tile each
], ids=lambda c: "x".join(map(str, c[:7])))
def test_short_sequences_whose_heads_share_keys(case, weight):
    """Up to 64 tokens of many heads, forward and backward take a group's queries as rows of one tile; each row
    and column then has its own head's weight."""
    B, T, S, H, Hk, d, dv, causal, start, lengths = case
    q, k, v, lam, dout = arrays(B, T, S, H, Hk, d, dv, T + S + 2)
    lam *= np.float32(weight)
    val, tol = reference(q, k, v, lam, dout, d ** -0.5, causal, start, lengths)
    check(call(q, k, v, lam, dout, causal=causal, query_start=start, lengths=lengths), val, tol)


@pytest.mark.parametrize("shape", [(50, 43, 43, 3, 1, 64, 128), (2, 43, 70, 3, 1, 40, 64)], ids=["shared", "own"])
def test_each_gradient_alone(shape):
    """Whichever inputs want a gradient, it is the one that all of them get together."""
    import tynx_b200 as tx

    q, k, v, lam, dout = arrays(*shape, 31)
    kw = dict(causal=True, query_start=0)
    together = call(q, k, v, lam, dout, lengths=None, **kw)[1:]
    for wanted in range(4):
        leaves = [tx.Tensor(a, requires_grad=i == wanted) for i, a in enumerate((q, k, v, lam))]
        tx.nn.functional.differential_attention(*leaves, **kw).backward(tx.Tensor(dout))
        for i, t in enumerate(leaves):
            assert (t.grad is None) == (i != wanted)
        np.testing.assert_array_equal(leaves[wanted].grad.numpy(), together[wanted].numpy())


def test_what_lies_behind_a_length_is_not_read():
    q, k, v, lam, dout = arrays(2, 70, 150, 2, 1, 64, 128, 5)
    lengths = [149, 70]
    kw = dict(causal=False, query_start=0, lengths=lengths)
    clean = call(q, k, v, lam, dout, **kw)
    for b, n in enumerate(lengths):
        k[b, n:] = np.nan
        v[b, n:] = np.inf
    for a, b in zip(clean, call(q, k, v, lam, dout, **kw)):
        np.testing.assert_array_equal(a.numpy(), b.numpy())


def test_queries_without_keys_give_zeros():
    q, k, v, lam, dout = arrays(2, 6, 4, 2, 2, 16, 32, 6)
    got = call(q, k, v, lam, dout, causal=True, query_start=None, lengths=None)  # the first two see nothing
    np.testing.assert_array_equal(got[0].numpy()[:, :2], 0.0)
    np.testing.assert_array_equal(got[1].numpy()[:, :2], 0.0)
    got = call(q, k, v, lam, dout, causal=False, query_start=None, lengths=[0, 0])
    for t in got:
        np.testing.assert_array_equal(t.numpy(), 0.0)


def test_no_keys_at_all():
    q, k, v, lam, dout = arrays(2, 3, 0, 2, 2, 16, 32, 7)
    for t in call(q, k, v, lam, dout, causal=False, query_start=None, lengths=None):
        np.testing.assert_array_equal(t.numpy(), 0.0)


def test_large_scores_stay_finite():
    """Scores of several hundred: the running maximum keeps every exponential at most 1."""
    q, k, v, lam, dout = arrays(1, 140, 300, 2, 2, 64, 128, 8)
    q *= 40.0
    got = call(q, k, v, lam, dout, causal=True, query_start=160, lengths=None)
    val, tol = reference(q, k, v, lam, dout, 0.125, True, 160, None)
    for g, w, t in zip(got, val, tol):
        assert np.isfinite(g.numpy()).all()
        assert np.all(np.abs(g.numpy() - w) <= 1.1 * t + 1e-30)


@pytest.mark.parametrize("sizes", [(1e15, 1e-15), (1e-12, 1e-10), (1e18, 1e12), (1e-25, 1e8)])
def test_any_magnitude(sizes):
    """Powers of two a tile carry the operands' and gradients' magnitudes."""
    q, k, v, lam, dout = arrays(1, 150, 150, 2, 1, 64, 128, 20)
    q, k, v, dout = q * 1e10, k * 1e-10, v * sizes[0], dout * sizes[1]
    q, k, v, dout = (a.astype(np.float32) for a in (q, k, v, dout))
    val, tol = reference(q, k, v, lam, dout, 0.125, True, 0, None)
    got = call(q, k, v, lam, dout, causal=True, query_start=0, lengths=None)
    for name, g, w, t in zip(("out", "dq", "dk", "dv", "dlam"), got, val, tol):
        g = g.numpy().astype(np.float64)
        # fp32 ends at 3.4e38.  A bound is at least E = 1.1e-5 of the magnitudes that its sum adds, so
        # where it passes 1e33 they pass 9e37 and the sum may leave the range (1e18 * 1e12 * 1e10 does).
        inside = t <= 1e33
        if name != "dk":
            assert inside.all(), name
        g, w, t = g[inside], w[inside], t[inside]
        assert np.isfinite(g).all(), name
        assert np.all(np.abs(g - w) <= 1.1 * t + 1e-37), name
        assert np.linalg.norm(g - w) <= 1e-5 * np.linalg.norm(w) + 1e-37, name


@pytest.mark.parametrize("lam_size,scale", [(0.0, 0.125), (-3.0, 0.125), (100.0, 0.05), (0.5, -0.2), (0.5, 0.0)])
def test_any_weight_and_scale(lam_size, scale):
    q, k, v, lam, dout = arrays(2, 70, 140, 4, 2, 32, 64, 21)
    lam = (lam * lam_size).astype(np.float32)
    val, tol = reference(q, k, v, lam, dout, scale, False, 0, [140, 77])
    check(call(q, k, v, lam, dout, causal=False, query_start=0, lengths=[140, 77], scale=scale), val, tol)


def test_rows_of_very_different_size():
    """A tile's power of two follows its largest row: rows 2^10 smaller keep their precision."""
    q, k, v, lam, dout = arrays(1, 140, 260, 2, 2, 64, 128, 22)
    q[0, 3] *= 30.0
    v[0, 100:110] *= 1000.0
    dout[0, 20] *= 1000.0
    k[0, 200:] *= 0.01
    val, tol = reference(q, k, v, lam, dout, 0.125, True, 120, None)
    check(call(q, k, v, lam, dout, causal=True, query_start=120, lengths=None), val, tol)


def test_one_tensor_as_queries_and_keys_and_partial_gradients():
    import tynx_b200 as tx

    F = tx.nn.functional
    q, _, v, lam, dout = arrays(1, 40, 40, 2, 2, 16, 32, 23)
    val = reference(q, q, v, lam, dout, 0.25, True, 0, None)[0]
    Q, V, L = tx.Tensor(q, requires_grad=True), tx.Tensor(v), tx.Tensor(lam)
    F.differential_attention(Q, Q, V, L, causal=True).backward(tx.Tensor(dout))
    want = val[1] + val[2]
    assert np.linalg.norm(Q.grad.numpy() - want) <= 2e-5 * np.linalg.norm(want) and V.grad is None and L.grad is None
    K = tx.Tensor(q)
    for i, (which, w) in enumerate(((V, val[3]), (L, val[4]))):  # each gradient wanted alone
        Q2 = tx.Tensor(q)
        which.requires_grad_()
        F.differential_attention(Q2, K, V, L, causal=True).backward(tx.Tensor(dout))
        assert np.linalg.norm(which.grad.numpy() - w) <= 1e-5 * np.linalg.norm(w), i
        which.requires_grad_(False)


def test_captured_steps_beside_an_eager_graph():
    """Two captured steps replayed in turn, while an eager graph of the same leaves is alive."""
    import tynx_b200 as tx

    F = tx.nn.functional
    sets = [arrays(1, 50, 90, 2, 1, 64, 128, s) for s in (30, 31)]
    leaves = [tx.Tensor(a, requires_grad=True) for a in sets[0][:4]]
    waiting = F.differential_attention(*leaves, causal=True)

    def step(q, k, v, lam, dout):
        q, k, v, lam = (t.detach().requires_grad_() for t in (q, k, v, lam))
        out = F.differential_attention(q, k, v, lam, causal=True)
        out.backward(dout)
        return [out.detach(), q.grad, k.grad, v.grad, lam.grad]

    def other(q, k, v, lam, dout):
        return [t * 2.0 for t in step(q, k, v, lam, dout)]

    first, second = tx.compile(step, fullgraph=True), tx.compile(other, fullgraph=True)
    for _ in range(2):
        for a in sets:
            tensors = [tx.Tensor(x) for x in a]
            eager = step(*tensors)
            for x, y, z in zip(first(*tensors), second(*tensors), eager):
                np.testing.assert_array_equal(x.numpy(), z.numpy())
                np.testing.assert_array_equal(y.numpy(), 2.0 * z.numpy())
    waiting.backward(tx.Tensor(sets[0][4]))
    for leaf, g in zip(leaves, step(*[tx.Tensor(x) for x in sets[0]])[1:]):
        np.testing.assert_array_equal(leaf.grad.numpy(), g.numpy())


def test_many_sequences():
    """More (sequence, head) pairs than a grid's second axis holds."""
    import tynx_b200 as tx

    q, k, v, lam, dout = arrays(9000, 1, 3, 8, 8, 4, 4, 24)
    with tx.no_grad():
        out = tx.nn.functional.differential_attention(*(tx.Tensor(a) for a in (q, k, v, lam))).numpy()
    for b in (0, 4321, 8999):
        val, tol = reference(q[b:b + 1], k[b:b + 1], v[b:b + 1], lam, dout[b:b + 1], 0.5, False, 0, None)
        assert np.all(np.abs(out[b:b + 1] - val[0]) <= 1.1 * tol[0] + 1e-30)


@pytest.mark.parametrize("queries", [1, 40])
def test_offsets_past_32_bits(queries):
    """The last sequence of a cache of 2.4e9 key elements gives what it gives alone."""
    import torch

    import tynx_b200 as tx

    gen = torch.Generator(device="cuda")
    gen.manual_seed(5)
    B, S, H, d, dv = 3, 100000, 64, 64, 8
    k = torch.randn(B, S, 2 * H, d, generator=gen, device="cuda")
    v = torch.randn(B, S, H, dv, generator=gen, device="cuda")
    q = torch.randn(B, queries, 2 * H, d, generator=gen, device="cuda")
    lam = torch.rand(H, generator=gen, device="cuda")
    assert k.numel() > 2**31
    F = tx.nn.functional
    L = tx.from_dlpack(lam)
    whole = F.differential_attention(tx.from_dlpack(q), tx.from_dlpack(k), tx.from_dlpack(v), L).numpy()
    alone = F.differential_attention(*(tx.from_dlpack(t[2:].contiguous()) for t in (q, k, v)), L).numpy()
    # the keys may be shared out over other ranges, so sums have another order: each is within E of its
    # terms' magnitudes, which add to (1 + lam) mean|v| < 2, of the exact value
    assert np.abs(whole[2:] - alone).max() <= 2 * E * 2
    for h in (0, 63):
        kk, vv, qq = k[2, :, 2 * h:2 * h + 2].double(), v[2, :, h].double(), q[2, :, 2 * h:2 * h + 2].double()
        a = torch.softmax(torch.einsum("tmd,smd->mts", qq, kk) / 8.0, -1)
        want = (a[0] @ vv - lam[h].double() * (a[1] @ vv)).cpu().numpy()
        assert np.linalg.norm(whole[2, :, h] - want) <= 1e-5 * np.linalg.norm(want)


def test_lengths_outside_the_keys_raise():
    import tynx_b200 as tx

    q, k, v, lam, _ = (tx.Tensor(a) for a in arrays(2, 3, 5, 2, 2, 16, 32, 9))
    for bad in ([5, 6], [-1, 5]):
        tx.nn.functional.differential_attention(q, k, v, lam, key_lengths=tx.Tensor(np.array(bad)))
        with pytest.raises(IndexError):
            tx.synchronize()
    tx.synchronize()


def test_gradient_agrees_with_differences():
    import tynx_b200 as tx

    data = list(arrays(1, 4, 5, 2, 1, 8, 6, 10))
    dout = data.pop().astype(np.float64)
    F = tx.nn.functional

    def value(a):
        with tx.no_grad():
            return float((F.differential_attention(*(tx.Tensor(x) for x in a), causal=True).numpy() * dout).sum())

    grads = call(*data, dout.astype(np.float32), causal=True, query_start=None, lengths=None)[1:]
    rng = np.random.default_rng(11)
    for i, g in enumerate(grads):
        way = rng.standard_normal(data[i].shape).astype(np.float32)
        h = 1e-2
        plus, minus = ([a + (h * s * way if j == i else 0) for j, a in enumerate(data)] for s in (1, -1))
        slope = (value(plus) - value(minus)) / (2 * h)
        # third differences h^2 / 6, and 1e-6 of the value over 2 h
        assert abs(slope - float((g.numpy() * way).sum())) <= 2e-3 * max(1.0, np.abs(g.numpy() * way).sum())


def test_same_inputs_give_the_same_bits():
    q, k, v, lam, dout = arrays(2, 150, 400, 4, 2, 64, 128, 12)
    kw = dict(causal=True, query_start=250, lengths=[400, 333])
    for a, b in zip(call(q, k, v, lam, dout, **kw), call(q, k, v, lam, dout, **kw)):
        np.testing.assert_array_equal(a.numpy(), b.numpy())


@pytest.mark.parametrize("shape", [
    (8, 1, 700, 4, 2, 64, 128),      # few queries, joined
    (2, 40, 2000, 4, 2, 64, 128),    # ranges of keys, joined
    (40, 50, 50, 4, 2, 64, 128),     # a group's heads in one tile
    (2, 300, 300, 6, 1, 40, 72),     # key blocks of single heads, summed
], ids=lambda c: "x".join(map(str, c)))
def test_calls_close_behind_one_another(shape):
    """Kernels of a call start under the ends of one another; results are those of calls far apart."""
    import tynx_b200 as tx

    sets, want = [arrays(*shape, 50 + i) for i in range(3)], []
    for a in sets:
        got = call(*a, causal=True, lengths=None)
        tx.synchronize()
        want.append([t.numpy() for t in got])
    many = [call(*sets[i % 3], causal=True, lengths=None) for i in range(24)]
    with tx.no_grad():
        tensors = [[tx.Tensor(x) for x in a[:4]] for a in sets]
        plain = [tx.nn.functional.differential_attention(*tensors[i % 3], causal=True) for i in range(24)]
    for i, got in enumerate(many):
        for g, w in zip(got, want[i % 3]):
            np.testing.assert_array_equal(g.numpy(), w)
        np.testing.assert_array_equal(plain[i].numpy(), plain[i % 3].numpy())


def test_layer_of_all_three_trains_and_replays():
    """Projections, norms with rotation, differential attention and a loss, eager and as a
    captured step replayed on other inputs, against each other and the 64-bit composition."""
    import tynx_b200 as tx

    F = tx.nn.functional
    B, T, E_, H, Hk, d, dv = 2, 37, 48, 4, 2, 16, 32
    rng = np.random.default_rng(13)
    shapes = [(E_, 2 * H * d), (E_, 2 * Hk * d), (E_, Hk * dv)]
    weights = [rng.standard_normal(s).astype(np.float32) / 7 for s in shapes] + \
        [np.ones(d, np.float32), np.ones(d, np.float32), np.full(H, 0.5, np.float32)]
    params = [tx.Tensor(w, requires_grad=True) for w in weights]
    rotary = tx.nn.Rotary(d)
    tx.set_math_mode("3xtf32")
    try:
        def step(x, y):
            for p in params:
                p.grad = None
            q = (x @ params[0]).reshape(B, T, 2 * H, d)
            k = (x @ params[1]).reshape(B, T, 2 * Hk, d)
            v = (x @ params[2]).reshape(B, T, Hk, dv)
            q, k = F.qk_norm_rotary(q, k, params[3], params[4], rotary)
            out = F.differential_attention(q, k, v, params[5], causal=True)
            loss = F.mse_loss(out, y)
            loss.backward()
            return [loss] + [p.grad for p in params]

        compiled = tx.compile(step, fullgraph=True)
        for seed in (0, 1, 2):
            r = np.random.default_rng(seed)
            x = tx.Tensor(r.standard_normal((B * T, E_)).astype(np.float32))
            y = tx.Tensor(r.standard_normal((B, T, H, dv)).astype(np.float32))
            replayed = [t.numpy() for t in compiled(x, y)]
            eager = [t.numpy() for t in step(x, y)]
            for a, b in zip(replayed, eager):
                np.testing.assert_array_equal(a, b)
        assert compiled.replay_count == 2
        # the 64-bit composition of the last step
        from tests.test_gpu_rotary import norm_reference, turned  # noqa: F401

        x64, y64 = x.numpy().astype(np.float64), y.numpy().astype(np.float64)
        q, k, v = (x64 @ w for w in weights[:3])
        q, k, v = q.reshape(B, T, 2 * H, d), k.reshape(B, T, 2 * Hk, d), v.reshape(B, T, Hk, dv)
        positions = np.broadcast_to(np.arange(T), (B, T))
        qn, kn = (norm_reference(a, np.ones(d), rotary, positions, 1e-6, np.zeros_like(a))[0] for a in (q, k))
        out = reference(qn, kn, v, weights[5], np.zeros((B, T, H, dv)), d ** -0.5, True, 0, None)[0][0]
        dout = 2 * (out - y64) / out.size
        val = reference(qn, kn, v, weights[5], dout, d ** -0.5, True, 0, None)[0]
        dq = norm_reference(q, np.ones(d), rotary, positions, 1e-6, val[1])
        dk = norm_reference(k, np.ones(d), rotary, positions, 1e-6, val[2])
        want = [((out - y64) ** 2).mean().reshape(1), x64.T @ dq[1].reshape(B * T, -1), x64.T @ dk[1].reshape(B * T, -1),
                x64.T @ val[3].reshape(B * T, -1), dq[2], dk[2], val[4]]
        for name, a, b in zip(("loss", "wq", "wk", "wv", "qw", "kw", "lam"), eager, want):
            # a chain of five stages of 1e-5 each
            assert np.linalg.norm(a - b) <= 5e-5 * np.linalg.norm(b), (name, np.linalg.norm(a - b) / np.linalg.norm(b))
    finally:
        tx.set_math_mode("tf32")
