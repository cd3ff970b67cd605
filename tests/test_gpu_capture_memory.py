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


def test_tensors_dropped_on_other_threads():
    """Whichever thread drops the last reference, or collects garbage, the allocator stays whole."""
    import queue
    import threading

    import tynx_b200 as tx

    dropped = queue.Queue()

    def drop():
        while dropped.get() is not None:
            pass

    threads = [threading.Thread(target=drop) for _ in range(4)]
    for thread in threads:
        thread.start()
    sizes = [1 << 10, 1 << 12, 1 << 16]
    compiled = tx.compile(lambda a: a * 2.0, fullgraph=True)
    wrong = 0
    for i in range(6000):
        t = tx.ones(sizes[i % 3]) * float(i)
        u = compiled(t)
        v = u + 1.0
        if i % 100 == 99:
            wrong += int((v.numpy() != 2.0 * i + 1.0).any())
        for x in (t, u, v):
            dropped.put(x)
        del t, u, v, x
    for _ in threads:
        dropped.put(None)
    for thread in threads:
        thread.join()
    assert wrong == 0
    held = [tx.ones(1 << 12) for _ in range(200)]
    assert len({t.ptr for t in held}) == 200
