"""How long memory that crosses to another library, or from one, stays out of use."""

import gc

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("borrowers", [1, 3])
def test_lent_memory_that_a_captured_step_let_go(borrowers):
    """A captured step reads a lent tensor and drops it: replays read it whoever lets go of it afterwards."""
    import torch

    import tynx_b200 as tx

    box = [tx.ones(1 << 18)]
    there = [torch.from_dlpack(box[0]) for _ in range(borrowers)]
    box[0].numpy()

    def step(a):
        return a + box.pop()

    compiled = tx.compile(step, fullgraph=True)
    zero = tx.zeros(1 << 18)
    np.testing.assert_array_equal(compiled(zero).numpy(), 1.0)
    assert not box
    while there:
        there.pop()
        gc.collect()
        others = [tx.Tensor(np.full(1 << 18, 7.0, np.float32)) for _ in range(4)]
        np.testing.assert_array_equal(compiled(zero).numpy(), 1.0)
        del others


def test_lent_memory_that_was_let_go_outside_a_capture_is_used_again():
    import torch

    import tynx_b200 as tx

    before = tx.ones(5_000_001)
    at = before.ptr
    there = torch.from_dlpack(before)
    del before
    assert tx.ones(5_000_001).ptr != at
    del there
    gc.collect()
    held = [tx.ones(5_000_001) for _ in range(3)]
    assert at in [t.ptr for t in held]


def test_a_copy_is_a_copy():
    import torch

    import tynx_b200 as tx

    mine = tx.Tensor(np.arange(6, dtype=np.float32))
    there = torch.from_dlpack(mine, copy=True)
    there += 1.0
    torch.cuda.synchronize()
    np.testing.assert_array_equal(mine.numpy(), np.arange(6))
    np.testing.assert_array_equal(there.cpu().numpy(), 1 + np.arange(6))
    alias = torch.from_dlpack(mine, copy=False)
    alias += 1.0
    torch.cuda.synchronize()
    np.testing.assert_array_equal(mine.numpy(), 1 + np.arange(6))
    named = torch.from_dlpack(mine, device="cuda")
    assert named.data_ptr() == mine.ptr
    parameter = tx.ones(3).requires_grad_()
    with pytest.raises(BufferError, match="detach"):
        parameter.__dlpack__(copy=True)
    kept = torch.utils.dlpack.from_dlpack(mine.reshape(2, 3).__dlpack__(stream=1, max_version=(1, 0), copy=True,
                                                                       dl_device=(2, 0)))
    del mine, alias, named
    gc.collect()
    spoil = [tx.zeros(6) for _ in range(4)]
    tx.synchronize()
    np.testing.assert_array_equal(kept.cpu().numpy(), 1 + np.arange(6).reshape(2, 3))
    del spoil


def test_borrowed_memory_that_a_captured_step_let_go():
    """It stays with the captured graph that reads it, and goes back with it."""
    import torch

    import tynx_b200 as tx

    n = 3 << 20
    box = [tx.from_dlpack(torch.ones(n, device="cuda"))]

    def step(a):
        return a + box.pop()

    compiled = tx.compile(step, fullgraph=True)
    zero = tx.zeros(n)
    np.testing.assert_array_equal(compiled(zero).numpy(), 1.0)
    assert not box
    gc.collect()
    tx.from_dlpack(torch.zeros(1, device="cuda"))
    others = [torch.full((n,), 7.0, device="cuda") for _ in range(3)]
    torch.cuda.synchronize()
    np.testing.assert_array_equal(compiled(zero).numpy(), 1.0)
    del others
    gc.collect()
    held = torch.cuda.memory_allocated()
    compiled.clear_cache()
    gc.collect()
    assert torch.cuda.memory_allocated() <= held - 4 * n


def test_borrowed_memory_let_go_in_a_step_that_was_not_captured():
    """A body that cannot be captured runs eagerly; what it let go while it was being recorded goes back."""
    import torch

    import tynx_b200 as tx

    n = 3 << 20
    gc.collect()
    free = torch.cuda.memory_allocated()
    box = [tx.from_dlpack(torch.ones(n, device="cuda")) for _ in range(2)]

    def step(a):
        out = a + box.pop()
        return out * float(out.sum().item())

    compiled = tx.compile(step)
    with pytest.warns(RuntimeWarning, match="eager"):
        out = compiled(tx.zeros(n))
    np.testing.assert_array_equal(out.numpy(), float(n))
    assert not box
    gc.collect()
    assert torch.cuda.memory_allocated() <= free


def test_borrowed_memory_let_go_on_another_thread():
    import threading

    import torch

    import tynx_b200 as tx

    n = 3 << 20
    torch.cuda.synchronize()
    gc.collect()
    free = torch.cuda.memory_allocated()
    box = [tx.from_dlpack(torch.ones(n, device="cuda"))]
    assert torch.cuda.memory_allocated() > free
    thread = threading.Thread(target=box.clear)
    thread.start()
    thread.join()
    gc.collect()
    assert torch.cuda.memory_allocated() <= free
    np.testing.assert_array_equal(tx.from_dlpack(torch.ones(3, device="cuda")).numpy(), 1.0)
