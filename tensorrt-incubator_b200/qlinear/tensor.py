"""Tensor plumbing between torch (device memory, streams) and the C ABI."""
from __future__ import annotations

import functools
import math

import torch

from . import _lib
from . import dtypes as dt


class Int4Tensor:
    """Signed 4-bit values, two per byte with the first element in the low nibble (the layout the
    reference gives TensorRT: tensorrt/lib/Target/TensorRTEncodingOpInterface/NetworkEncoder.cpp:552-570).
    `packed` is a flat uint8 tensor of ceil(numel / 2) bytes; `shape` is the logical shape."""

    dtype = dt.int4

    def __init__(self, packed: torch.Tensor, shape):
        self.shape = tuple(int(s) for s in shape)
        n = math.prod(self.shape)
        assert packed.dtype == torch.uint8 and packed.numel() == (n + 1) // 2
        self.packed = packed.contiguous()

    @property
    def device(self):
        return self.packed.device

    def numel(self) -> int:
        return math.prod(self.shape)

    def unpack(self) -> torch.Tensor:
        """int8 tensor of the logical shape (a host-side convenience for tests)."""
        p = self.packed.to(torch.int16)
        lo = p & 0xF
        hi = (p >> 4) & 0xF
        v = torch.stack([lo, hi], dim=1).reshape(-1)[: self.numel()]
        return (((v ^ 8) - 8).to(torch.int8)).reshape(self.shape)

    @staticmethod
    def pack(values: torch.Tensor) -> "Int4Tensor":
        v = values.reshape(-1).to(torch.int16) & 0xF
        if v.numel() % 2:
            v = torch.cat([v, v.new_zeros(1)])
        packed = (v[0::2] | (v[1::2] << 4)).to(torch.uint8)
        return Int4Tensor(packed, values.shape)


class Float4Tensor:
    """e2m1 values, two per byte with the first element in the low nibble; `packed` is a flat uint8 tensor of
    numel / 2 bytes, `shape` the logical shape.  The scales beside it say which format it belongs to: e4m3 for each 16 values
    along the last dimension (NVFP4, dynamic_quantize), or e8m0 for each 32 (MXFP4, quantize_mxfp4)."""

    dtype = dt.float4
    _VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)

    def __init__(self, packed: torch.Tensor, shape):
        self.shape = tuple(map(int, shape))
        assert packed.dtype == torch.uint8 and packed.numel() * 2 == math.prod(self.shape)
        self.packed = packed.contiguous()

    @staticmethod
    def empty(shape, device) -> "Float4Tensor":
        """Room for values of `shape` (a tuple with an even number of them)."""
        t = Float4Tensor.__new__(Float4Tensor)
        t.shape, t.packed = shape, empty((math.prod(shape) // 2,), torch.uint8, device)
        return t

    @property
    def device(self):
        return self.packed.device

    def numel(self) -> int:
        return math.prod(self.shape)

    def unpack(self) -> torch.Tensor:
        """float32 tensor of the logical shape (a host-side convenience for tests)."""
        p = self.packed.to(torch.int64)
        codes = torch.stack([p & 0xF, (p >> 4) & 0xF], dim=1).reshape(-1)
        lut = torch.tensor(self._VALUES + tuple(-v for v in self._VALUES), dtype=torch.float32, device=codes.device)
        return lut[codes].reshape(self.shape)


def dtype_of(t) -> dt.dtype:
    if isinstance(t, Float4Tensor):
        return dt.float4
    if isinstance(t, Int4Tensor):
        return dt.int4
    return dt.from_torch(t.dtype)


@functools.lru_cache(maxsize=1024)
def _view_of(dtype, shape) -> bytes:
    """The bytes of a QlTensor of this type (torch's, or the ABI's number) and shape, without its address."""
    return bytes(_lib.make_tensor(None, dtype if isinstance(dtype, int) else dt.from_torch(dtype).code, shape))


def ql_view(t) -> _lib.QlTensor:
    """QlTensor over a CUDA torch tensor or Int4Tensor (no copy; the caller keeps `t` alive).  Made from the bytes of its kind:
    0.8 us, 1.8 field by field."""
    if isinstance(t, torch.Tensor):
        if not t.is_contiguous():
            raise _lib.QlError(_lib.ERR_INVALID_ARGUMENT, "tensors must be contiguous (dense row-major)")
        v = _lib.QlTensor.from_buffer_copy(_view_of(t.dtype, t.shape))
        v.data = t.data_ptr()
    else:
        v = _lib.QlTensor.from_buffer_copy(_view_of(_lib.I4 if isinstance(t, Int4Tensor) else _lib.F4E2M1, t.shape))
        v.data = t.packed.data_ptr()
    return v


@functools.lru_cache(maxsize=1024)
def _dense_strides(shape):
    strides, n = [], 1
    for s in reversed(shape):
        strides.append(n)
        n *= max(s, 1)
    return tuple(reversed(strides))


def empty(shape, dtype, device) -> torch.Tensor:
    """torch.empty of a tuple's shape; with the strides given the allocation takes 1.7 us, without 2.6."""
    return torch.empty_strided(shape, _dense_strides(shape), dtype=dtype, device=device)


def require_cuda(t, what: str) -> None:
    dev = t.device
    if dev.type != "cuda":
        raise _lib.QlError(_lib.ERR_NO_DEVICE, f"{what} must live in GPU memory (got {dev}); there is no CPU path")


def current_stream(device) -> int:
    """The handle of `device`'s current stream (what torch.cuda.current_stream(device).cuda_stream is, without building the
    stream object: 0.1 us instead of 3 on every launch)."""
    index = device.index if isinstance(device, torch.device) else None
    if index is None:
        return torch.cuda.current_stream(device).cuda_stream
    return torch._C._cuda_getCurrentRawStream(index)


def empty_quantized(shape, qdtype: dt.dtype, device):
    if qdtype is dt.int4:
        n = math.prod(shape)
        return Int4Tensor(torch.empty((n + 1) // 2, dtype=torch.uint8, device=device), shape)
    return torch.empty(tuple(shape), dtype=qdtype.torch, device=device)


def call_on(device, fn, *args, same_device=()) -> None:
    """fn(*args, the current stream of `device`) with `device` current, whichever device was; every tensor of
    `same_device` has to live there."""
    for t in same_device:
        if t.device != device:
            raise _lib.QlError(_lib.ERR_INVALID_ARGUMENT, f"tensors must live on one device, got {device} and {t.device}")
    index = device.index
    if index is None or index == torch._C._cuda_getDevice():   # what torch.cuda.current_device() returns, without its start-up check
        rc = fn(*args, current_stream(device))
        if rc != _lib.OK:
            _lib.check(rc)
    else:
        with torch.cuda.device(device):
            _lib.check(fn(*args, current_stream(device)))
