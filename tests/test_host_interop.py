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


class _Library:
    """Stands in for the engine: notes what is given back."""

    def __init__(self):
        self.given = []

    def tx_dlpack_give_back(self, handle, managed):
        self.given.append((handle, managed))
        return 0


@pytest.mark.parametrize("capturing", [False, True])
def test_borrowed_memory_goes_back_whatever_thread_lets_go(monkeypatch, capturing):
    """The context belongs to another thread: the memory is given back at once, not kept for a later import."""
    from tynx_b200 import interop

    library = _Library()
    monkeypatch.setattr(interop, "lib", library)
    ctx = SimpleNamespace(index=0, handle=7, owner=-1, capturing=capturing)
    interop._Borrowed(ctx, 16, 4096, 99).__del__()
    assert library.given == [(7, 99)]


@pytest.mark.parametrize("capturing", [False, True])
def test_an_import_after_memory_that_another_thread_owns(monkeypatch, capturing):
    """An import returns, whatever was let go before it on a context that captures or is another thread's."""
    import threading

    from tynx_b200 import interop

    monkeypatch.setattr(interop, "lib", _Library())
    interop._Borrowed(SimpleNamespace(index=1, handle=7, owner=-1, capturing=capturing), 16, 4096, 99).__del__()

    class Reached(Exception):
        pass

    class Source:
        def __dlpack_device__(self):
            return (2, 0)

        def __dlpack__(self, stream):
            raise Reached

    own = SimpleNamespace(index=0, handle=8, capturing=False, check=lambda *a: None)
    monkeypatch.setattr(interop, "context", lambda device: own)
    interop.lib.tx_stream = lambda *a: 0
    results = []

    def call():
        try:
            interop.from_dlpack(Source())
        except Reached:
            results.append(True)

    thread = threading.Thread(target=call, daemon=True)
    thread.start()
    thread.join(20)
    assert results == [True]
