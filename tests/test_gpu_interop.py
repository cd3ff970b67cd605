"""Zero-copy exchange with torch in both directions."""

import gc

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def test_both_directions_share_memory():
    import torch

    import tynx_b200 as tx

    for array in (np.arange(12, dtype=np.float32).reshape(3, 4), np.arange(6), np.array([True, False]),
                  np.zeros((2, 0, 3), np.float32)):
        there = torch.from_dlpack(tx.Tensor(array))
        np.testing.assert_array_equal(there.cpu().numpy(), array)
        back = tx.from_dlpack(there)
        assert back.shape == array.shape
        np.testing.assert_array_equal(back.numpy(), array)
    t = torch.zeros(5, device="cuda")
    mine = tx.from_dlpack(t)
    t += 2.0
    torch.cuda.synchronize()
    np.testing.assert_array_equal(mine.numpy(), 2.0)
    assert torch.from_dlpack((mine * 3.0)).sum().item() == 30.0


def test_order_of_the_streams():
    """Results are handed over without a synchronisation on either side."""
    import torch

    import tynx_b200 as tx

    a = torch.randn(2048, 2048, device="cuda")
    for _ in range(20):
        b = a @ a  # queued on torch's stream
        mine = tx.from_dlpack(b)
        c = torch.from_dlpack(mine + 1.0)
        assert torch.equal(c, b + 1.0)


def test_lent_memory_is_reused_only_after_the_borrower():
    import torch

    import tynx_b200 as tx

    side = torch.cuda.Stream()
    for i in range(10):
        with torch.cuda.stream(side):
            there = torch.from_dlpack(tx.ones(1 << 20) * float(i))
            torch.cuda._sleep(2_000_000)  # the borrower reads late
            copy = there.clone()
            del there
        gc.collect()
        spoil = [tx.zeros(1 << 20) for _ in range(3)]
        side.synchronize()
        assert copy.min().item() == copy.max().item() == float(i)
        del spoil


def test_the_owner_may_go_first():
    import torch

    import tynx_b200 as tx

    mine = tx.ones(1000)
    there = torch.from_dlpack(mine)
    view = torch.from_dlpack(mine.reshape(10, 100))
    del mine
    others = [tx.zeros(1000) for _ in range(4)]
    tx.synchronize()
    assert there.sum().item() == 1000.0 and view.sum().item() == 1000.0
    del others


def test_operators_on_tensors_of_a_side_stream():
    """A tensor still being written on another stream is waited for, and the result handed back to that
    stream."""
    import torch

    import tynx_b200 as tx

    side = torch.cuda.Stream()
    rotary = tx.nn.Rotary(64)
    want = None
    for _ in range(5):
        with torch.cuda.stream(side):
            x = torch.ones(2, 300, 4, 64, device="cuda")
            torch.cuda._sleep(1_000_000)
            x *= 2.0
            y = torch.from_dlpack(tx.nn.functional.rotary_embedding(tx.from_dlpack(x), rotary))
            total = y.square().sum()
        side.synchronize()
        want = want or total.item()
        # a rotation keeps the sum of squares: 4 a value
        assert total.item() == want and abs(want - 4.0 * 2 * 300 * 4 * 64) < 1.0


def test_refusals():
    import torch

    import tynx_b200 as tx

    with pytest.raises(ValueError, match="contiguous"):
        tx.from_dlpack(torch.zeros(4, 6, device="cuda").t())
    with pytest.raises(ValueError, match="float32, int64 or bool"):
        tx.from_dlpack(torch.zeros(4, device="cuda", dtype=torch.float16))
    with pytest.raises(ValueError, match="CUDA tensors"):
        tx.from_dlpack(torch.zeros(4))
    with pytest.raises(BufferError, match="detach"):
        torch.from_dlpack(tx.ones(3).requires_grad_())
    with pytest.raises(ValueError, match="owns its memory"):
        tx.from_dlpack(torch.zeros(4, device="cuda")).__dlpack__()
    tx.ones(3).__dlpack__()  # a capsule that nobody takes ends its loan
    tx.synchronize()


def test_giving_memory_back_keeps_the_error():
    """A kernel's error is raised by the next synchronisation, also when borrowed memory went before it."""
    import torch

    import tynx_b200 as tx

    q, k, v = (tx.ones(1, 2, 2, 16), tx.ones(1, 4, 2, 16), tx.ones(1, 4, 1, 16))
    lengths = tx.from_dlpack(torch.tensor([9], device="cuda"))
    out = tx.nn.functional.differential_attention(q, k, v, tx.ones(1), key_lengths=lengths)
    del lengths
    gc.collect()
    with pytest.raises(IndexError):
        tx.synchronize()
    assert out.shape == (1, 2, 1, 16)
    tx.synchronize()


def test_backward_from_an_output_twice_and_from_its_input():
    """Roots may repeat, and one may lead to another: their gradients add."""
    import tynx_b200 as tx

    x = tx.ones(3).requires_grad_()
    y = x * 2.0
    z = y * 3.0
    one = tx.ones(3)
    tx.backward([y, z, y], [one, one, one])
    np.testing.assert_array_equal(x.grad.numpy(), 2.0 * (1 + 3 + 1))
    np.testing.assert_array_equal(one.numpy(), 1.0)
