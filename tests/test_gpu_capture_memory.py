"""Memory of captured graphs that are gone."""

import gc

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def test_a_late_release_names_no_other_tensor():
    """A captured step's tensors may be dropped after its graph's memory has gone back: a tensor that has got the
    address meanwhile keeps its block."""
    import tynx_b200 as tx

    kept = []

    def step(a):
        kept.append(a * 2.0)
        return kept[-1] + 1.0

    sizes = [1 << 18, 1 << 20, 16 << 20]
    for n in [1 << 10] + sizes:
        compiled = tx.compile(step, fullgraph=True)
        np.testing.assert_array_equal(compiled(tx.ones(n)).numpy(), 3.0)
        address = kept[0].ptr
        compiled.clear_cache()
        gc.collect()
        held = [tx.ones(sizes[i % 3]) for i in range(45)]
        assert address not in [t.ptr for t in held]
        kept.clear()
        gc.collect()
        again = [tx.zeros(s) for s in sizes]
        assert not {t.ptr for t in held} & {t.ptr for t in again}
        for t in held:
            np.testing.assert_array_equal(t.numpy(), 1.0)
        del held, again
