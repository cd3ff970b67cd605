"""The DLPack exchange's requests and refusals, without a GPU."""

from types import SimpleNamespace

import pytest


def on(index):
    """A Tensor whose memory no call reaches."""
    from tynx_b200 import Tensor

    t = object.__new__(Tensor)
    t._init(SimpleNamespace(ctx=SimpleNamespace(index=index)), 0, (3,), "float32")
    return t


@pytest.mark.parametrize("device", [(1, 0), (2, 1), (13, 0)])
def test_memory_of_another_device_is_refused(device):
    with pytest.raises(BufferError, match="device"):
        on(0).__dlpack__(dl_device=device)


def test_a_request_outside_the_protocol_is_refused():
    with pytest.raises(TypeError):
        on(0).__dlpack__(order="F")
