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


def _runtime():
    import ctypes

    import torch  # noqa: F401  (maps the runtime)

    with open("/proc/self/maps") as maps:
        path = next(line.split()[-1] for line in maps if "libcudart.so" in line)
    return ctypes.CDLL(path)


def test_a_borrower_whose_stream_is_gone():
    """Its memory is used again only after the work that the stream still had, without the stream's handle."""
    import ctypes

    import torch

    import tynx_b200 as tx

    runtime = _runtime()
    copy = torch.empty(1 << 20, device="cuda")
    for i in range(5):
        handle = ctypes.c_void_p()
        assert runtime.cudaStreamCreateWithFlags(ctypes.byref(handle), 1) == 0
        capsule = (tx.ones(1 << 20) * float(i)).__dlpack__(stream=handle.value)
        there = torch.utils.dlpack.from_dlpack(capsule)
        torch.cuda.synchronize()
        with torch.cuda.stream(torch.cuda.ExternalStream(handle.value)):
            torch.cuda._sleep(200_000_000)
            copy.copy_(there)
        del there
        assert runtime.cudaStreamDestroy(handle) == 0
        spoil = [tx.zeros(1 << 20) for _ in range(3)]
        tx.synchronize()
        torch.cuda.synchronize()
        assert copy.min().item() == copy.max().item() == float(i)
        del spoil


def test_a_borrower_that_captures():
    """What it lets go while its stream is recorded stays out of use; it cannot borrow meanwhile.  (A graph
    that reads what was borrowed on another stream has to keep it, as it has to keep its own memory.)"""
    import torch

    import tynx_b200 as tx
    from tynx_b200._native import CaptureError

    side = torch.cuda.Stream()
    mine = tx.ones(1 << 20)
    with torch.cuda.stream(side):
        box = [torch.from_dlpack(mine)]
    del mine
    copy = torch.zeros(1 << 20, device="cuda")
    other = tx.ones(5)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        with pytest.raises(CaptureError):
            torch.from_dlpack(other)
        copy.copy_(box.pop())
    gc.collect()
    spoil = [tx.Tensor(np.full(1 << 20, 7.0, np.float32)) for _ in range(3)]
    tx.synchronize()
    graph.replay()
    torch.cuda.synchronize()
    assert copy.min().item() == copy.max().item() == 1.0
    np.testing.assert_array_equal(torch.from_dlpack(other).cpu().numpy(), 1.0)
    del spoil


def test_one_stream_on_both_sides():
    """A loan on the context's own stream needs no event."""
    import torch

    import tynx_b200 as tx

    for i in range(20):
        there = torch.utils.dlpack.from_dlpack((tx.ones(4096) * float(i)).__dlpack__(stream=-1))
        tx.synchronize()
        assert there.sum().item() == 4096.0 * i
        again = tx.from_dlpack(tx.ones(16))
        np.testing.assert_array_equal((again + 1.0).numpy(), 2.0)


def test_the_default_stream_while_a_stream_beside_it_is_captured():
    """The legacy default stream takes no work then: loans wait, and the capture stays whole."""
    import ctypes

    import torch

    import tynx_b200 as tx
    from tynx_b200._native import CaptureError

    runtime = _runtime()
    warm = [tx.ones(4_000_001) for _ in range(4)]
    mine = warm.pop()
    at = mine.ptr
    there = torch.from_dlpack(mine)
    small = tx.ones(3)
    del mine, warm
    tx.synchronize()
    torch.cuda.synchronize()
    handle, graph = ctypes.c_void_p(), ctypes.c_void_p()
    assert runtime.cudaStreamCreate(ctypes.byref(handle)) == 0
    assert runtime.cudaStreamBeginCapture(handle, 2) == 0
    del there
    gc.collect()
    others = [tx.ones(4_000_001) for _ in range(3)]
    pointers = [t.ptr for t in others]
    refused = False
    try:
        torch.from_dlpack(small)
    except CaptureError:
        refused = True
    assert runtime.cudaStreamEndCapture(handle, ctypes.byref(graph)) == 0
    assert refused and at not in pointers
    held = tx.ones(4_000_001)
    assert held.ptr == at
    runtime.cudaGraphDestroy(graph)
    assert runtime.cudaStreamDestroy(handle) == 0
    np.testing.assert_array_equal(torch.from_dlpack(small).cpu().numpy(), 1.0)
    del others


def test_a_threads_default_stream_let_go_on_another_thread():
    """Its handle means another stream there: the borrower's work is waited for all the same."""
    import ctypes
    import threading

    import torch

    import tynx_b200 as tx

    runtime, own = _runtime(), ctypes.c_void_p(2)
    copy = torch.empty(1 << 20, device="cuda")
    side = torch.cuda.Stream()
    for i in range(5):
        box = [torch.utils.dlpack.from_dlpack((tx.ones(1 << 20) * float(i)).__dlpack__(stream=2))]
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            torch.cuda._sleep(200_000_000)
            late = torch.cuda.Event()
            late.record(side)
        assert runtime.cudaStreamWaitEvent(own, ctypes.c_void_p(late.cuda_event), 0) == 0
        assert runtime.cudaMemcpyAsync(ctypes.c_void_p(copy.data_ptr()), ctypes.c_void_p(box[0].data_ptr()),
                                       ctypes.c_size_t(4 << 20), 3, own) == 0
        thread = threading.Thread(target=box.clear)
        thread.start()
        thread.join()
        spoil = [tx.zeros(1 << 20) - 1.0 for _ in range(3)]
        assert runtime.cudaStreamSynchronize(own) == 0
        tx.synchronize()
        assert copy.min().item() == copy.max().item() == float(i)
        del spoil
