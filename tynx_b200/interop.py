"""Device tensors to and from other libraries of the process without a copy (DLPack).

``torch.from_dlpack(tensor)`` (or any consumer of the protocol) takes a
:class:`Tensor`'s memory through ``Tensor.__dlpack__``; :func:`from_dlpack` takes
another library's CUDA tensor.  Both directions are ordered on the streams of
both sides: work issued afterwards on the taker's stream sees the work that the
giver had issued.  A block that was lent is reused only after the borrower's
stream has passed the point where it let go of it.  A write through either side
is seen by both, also by a backward that kept the values.
"""

from __future__ import annotations

import ctypes as C

from . import _native as N
from ._core import Context, Device, Storage, Tensor, context
from ._native import CaptureError, lib

_CUDA = 2


class _DLTensor(C.Structure):
    _fields_ = [("data", C.c_void_p), ("device_type", C.c_int32), ("device_id", C.c_int32), ("ndim", C.c_int32),
                ("code", C.c_uint8), ("bits", C.c_uint8), ("lanes", C.c_uint16), ("shape", C.POINTER(C.c_int64)),
                ("strides", C.POINTER(C.c_int64)), ("byte_offset", C.c_uint64)]


_DTYPES = {(2, 32, 1): "float32", (0, 64, 1): "int64", (6, 8, 1): "bool"}
_SHAPES = [C.c_int64 * n for n in range(N.MAX_DIMS + 1)]
_NAME, _USED = b"dltensor", b"used_dltensor"

_api = C.pythonapi
_new = _api.PyCapsule_New
_new.restype, _new.argtypes = C.py_object, [C.c_void_p, C.c_char_p, C.c_void_p]
_valid = C.PYFUNCTYPE(C.c_int, C.c_void_p, C.c_char_p)(("PyCapsule_IsValid", _api))
_pointer = C.PYFUNCTYPE(C.c_void_p, C.c_void_p, C.c_char_p)(("PyCapsule_GetPointer", _api))
_rename = _api.PyCapsule_SetName
_rename.restype, _rename.argtypes = C.c_int, [C.py_object, C.c_char_p]
_take = _api.PyCapsule_GetPointer
_take.restype, _take.argtypes = C.c_void_p, [C.py_object, C.c_char_p]


@C.PYFUNCTYPE(None, C.c_void_p)
def _drop(capsule):
    """Ends the loan of a capsule that nobody took."""
    if _valid(capsule, _NAME):
        lib.tx_dlpack_release(_pointer(capsule, _NAME))


_drop_pointer = C.cast(_drop, C.c_void_p)


def export(tensor: Tensor, stream=None, device=None, copy=None):
    """The capsule behind ``Tensor.__dlpack__``; ``stream`` as the protocol has it
    for CUDA: None or 1 the legacy default stream, 2 the thread's default one, -1
    no ordering, otherwise a ``cudaStream_t``.  ``device`` is the (type, index) that
    the memory has to be on, ``copy`` True for memory of its own."""
    if tensor.requires_grad:
        raise BufferError("a Tensor that requires gradients cannot be exported; detach() it first")
    if stream == 0:
        raise ValueError("stream 0 is ambiguous in the DLPack protocol; use 1, 2 or a stream handle")
    if device is not None and tuple(map(int, device)) != tensor.__dlpack_device__():
        raise BufferError(f"a Tensor on {tensor.device} cannot be exported to DLPack device {tuple(map(int, device))}")
    if copy:
        tensor = tensor.clone()
    storage, shape = tensor._storage, tensor.shape
    ctx = storage.ctx
    if stream == -1:  # ordering with itself adds none
        own = C.c_void_p()
        ctx.check(lib.tx_stream(ctx.handle, C.byref(own)))
        stream = own.value
    ndim, data, cell = len(shape), storage.ptr, ctx.cell()
    code = lib.tx_dlpack_export(ctx.handle, data if storage.owned else None, data + tensor._offset,
                                N.DL_TYPES[tensor.dtype], _SHAPES[ndim](*shape), ndim, stream or 1, cell[1])
    managed = cell[0].value
    ctx.cells.append(cell)
    if code:
        ctx.check(code, "dlpack")
    return _new(managed, _NAME, _drop_pointer)


class _Borrowed(Storage):
    """Another library's memory; given back when the last Tensor on it goes, once
    the compute stream has passed the work issued on it (during a capture: with
    the captured graph, which may read it)."""

    __slots__ = ("managed",)

    def __init__(self, ctx: Context, nbytes: int, ptr: int, managed: int):
        super().__init__(ctx, nbytes, ptr=ptr, owned=False)
        self.managed = managed

    def __del__(self):
        managed, self.managed = getattr(self, "managed", None), None
        if managed:
            try:
                lib.tx_dlpack_give_back(self.ctx.handle, managed)  # whatever thread lets go
            except Exception:  # interpreter shutdown
                pass


def from_dlpack(source, device: Device | None = None) -> Tensor:
    """A Tensor on the memory of another library's CUDA tensor (float32, int64 or
    bool, dense row-major), without a copy.  Writes through either are seen by
    both; the source's memory is kept until the Tensor and its views are gone."""
    kind, index = source.__dlpack_device__()
    if int(kind) != _CUDA:
        raise ValueError(f"from_dlpack takes CUDA tensors, got device type {int(kind)}")
    if device is not None and device.index != index:
        raise ValueError(f"from_dlpack does not copy: the source is on cuda:{index}, not {device}")
    ctx = context(Device(f"cuda:{index}"))
    if ctx.capturing:
        raise CaptureError("from_dlpack is not allowed during a capture")
    stream = C.c_void_p()
    ctx.check(lib.tx_stream(ctx.handle, C.byref(stream)))
    capsule = source.__dlpack__(stream=stream.value)
    managed = _take(capsule, _NAME)
    t = C.cast(managed, C.POINTER(_DLTensor)).contents
    dtype = _DTYPES.get((t.code, t.bits, t.lanes))
    shape = tuple(t.shape[i] for i in range(t.ndim))
    if dtype is None:
        raise ValueError("from_dlpack takes float32, int64 or bool tensors, got DLPack type "
                         f"(code {t.code}, {t.bits} bits, {t.lanes} lanes)")
    if len(shape) > N.MAX_DIMS:
        raise ValueError(f"from_dlpack takes up to {N.MAX_DIMS} axes, got {len(shape)}")
    if t.strides and 0 not in shape:
        step = 1
        for size, stride in zip(reversed(shape), [t.strides[i] for i in reversed(range(t.ndim))]):
            if size != 1 and stride != step:
                raise ValueError("from_dlpack takes dense row-major tensors; make the source contiguous first")
            step *= size
    nbytes = t.bits // 8
    for size in shape:
        nbytes *= size
    if nbytes and ((t.data or 0) + t.byte_offset) % (t.bits // 8):
        raise ValueError("from_dlpack takes tensors aligned to their element size")
    _rename(capsule, _USED)  # from here on the structure is ours to release
    return Tensor._view(_Borrowed(ctx, nbytes, (t.data or 0) + t.byte_offset, managed), 0, shape, dtype)


__all__ = ["from_dlpack"]
