"""Allocations' results on the host side, without a GPU."""


def test_an_allocation_between_call_and_read(monkeypatch):
    """Another thread's allocation, or one that a finaliser makes, may come between an allocation and the
    read of its result: each has its own."""
    from tynx_b200 import _core

    inner = []

    class Library:
        count = 0

        def tx_alloc(self, handle, nbytes, out):
            self.count += 1
            out._obj.value = 4096 * self.count
            if self.count == 1:
                inner.append(_core.Storage(ctx, 8))
            return 0

        def tx_free(self, handle, ptr):
            return 0

    monkeypatch.setattr(_core, "lib", Library())
    ctx = object.__new__(_core.Context)
    ctx.handle = 1
    ctx.cells = []
    ctx._out = _core.C.c_void_p()
    ctx._out_ref = _core.C.byref(ctx._out)
    outer = _core.Storage(ctx, 8)
    got = outer.ptr, inner[0].ptr
    outer.ptr = inner[0].ptr = 0  # nothing for the engine to free
    assert got == (4096, 8192)
