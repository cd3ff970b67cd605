"""The per-head norms where nothing is added to the mean square, against 64-bit numpy.

Bounds as in test_gpu_rotary.py: they are relative to a row's or a sum's own terms and do not use eps.
"""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("eps", [0.0, 1e-60])  # the second vanishes in 32 bits
@pytest.mark.parametrize("batch,seq,heads,kv,dim,rot", [
    (1, 1, 1, 1, 8, 8), (3, 7, 5, 1, 40, 20), (2, 65, 6, 3, 96, 64), (1, 9, 32, 8, 256, 256), (1, 4096, 4, 4, 16, 16)])
def test_no_eps(batch, seq, heads, kv, dim, rot, eps):
    """The rows that fill up a block's last round take no part in the weights' gradients."""
    import tynx_b200 as tx
    from tests.test_gpu_rotary import close, norm_reference

    rng = np.random.default_rng(dim + seq)
    rotary = tx.nn.Rotary(rot)
    positions = np.broadcast_to(np.arange(seq), (batch, seq))
    q, dq = (rng.standard_normal((batch, seq, heads, dim)).astype(np.float32) for _ in range(2))
    k, dk = (rng.standard_normal((batch, seq, kv, dim)).astype(np.float32) for _ in range(2))
    qw, kw = (1 + 0.2 * rng.standard_normal(dim).astype(np.float32) for _ in range(2))
    leaves = [tx.Tensor(a, requires_grad=True) for a in (q, k, qw, kw)]
    outs = tx.nn.functional.qk_norm_rotary(*leaves, rotary, eps=eps)
    tx.backward(outs, [tx.Tensor(dq), tx.Tensor(dk)])
    for i, (x, w, dy) in enumerate(((q, qw, dq), (k, kw, dk))):
        y, dx, dw, size, total = norm_reference(x, w, rotary, positions, 0.0, dy)
        close(outs[i], y, 2e-6)
        close(leaves[i].grad, dx, 4e-6, size)
        close(leaves[i + 2].grad, dw, 1e-5, total)
