"""Microscaled 4-bit floating point (the OCP MX format MXFP4): e2m1 values in blocks of 32 along the last axis, one e8m0
scale (a power of two) per block.  Data are Float4Tensor, as dynamic_quantize's NVFP4 data are; scales are torch tensors of
torch.float8_e8m0fnu.  The reference has no such operator; NVFP4 (ops.dynamic_quantize) is its nearest relative."""
from __future__ import annotations

import ctypes
import functools

import torch

from . import _lib
from . import dtypes as dt
from .ops import QuantizeError
from .tensor import Float4Tensor, call_on, empty, ql_view, require_cuda

BLOCK = 32
_FLOATS = frozenset((torch.float32, torch.float16, torch.bfloat16))


def quantize_mxfp4(input: torch.Tensor):
    """(data, scales) of `input` [..., K] (float32, float16 or bfloat16; K a multiple of 32): scales[..., b] is
    2^(floor(log2 max|block b|) - 2), at least 2^-127, and data the block over its scale in e2m1, rounded half to even and
    saturated.  A block with an infinity or a NaN in it gets a NaN scale."""
    require_cuda(input, "input")
    if input.dtype not in _FLOATS:
        raise QuantizeError(f"Input does not have a valid dtype in quantize_mxfp4. input.dtype must be one of {dt.QUANTIZABLE_DTYPES}, got {input.dtype}")
    shape = tuple(input.shape)
    if not shape or shape[-1] % BLOCK:
        raise QuantizeError(f"the last dimension must be divisible by {BLOCK}, got shape {shape}.")
    x, device = input.contiguous(), input.device
    data = Float4Tensor.empty(shape, device)
    scales = empty(shape[:-1] + (shape[-1] // BLOCK,), torch.float8_e8m0fnu, device)
    call_on(device, _lib.lib().ql_quantize_mxfp4, ql_view(x), ql_view(data), ql_view(scales))
    return data, scales


def dequantize_mxfp4(data: Float4Tensor, scales: torch.Tensor, dtype: dt.dtype = dt.float32, out=None) -> torch.Tensor:
    """data * scales as `dtype` (float32, float16 or bfloat16): the inverse of quantize_mxfp4."""
    require_cuda(data, "data")
    require_cuda(scales, "scales")
    if dtype not in dt.QUANTIZABLE_DTYPES:
        raise QuantizeError(f"Unsupported data type in dequantize_mxfp4. Supported data types are: {dt.QUANTIZABLE_DTYPES}. Got dtype={dtype}")
    y = out if out is not None else empty(data.shape, dtype.torch, data.device)
    s = scales.contiguous()   # kept alive across the call: a view only borrows the pointer
    call_on(data.device, _lib.lib().ql_dequantize_mxfp4, ql_view(data), ql_view(s), ql_view(y), same_device=(s, y))
    return y


@functools.lru_cache(maxsize=256)
def _padding_bytes(a_shape, b_shape) -> int:
    """ql_gemm_mxfp4_workspace of operands whose scales are no 16-byte rows (it looks at addresses' alignment only), asked once
    per shape."""
    def operand(shape):
        return _lib.make_tensor(4, _lib.F4E2M1, shape), _lib.make_tensor(4, _lib.F8E8M0, (shape[0], shape[1] // BLOCK))
    size = ctypes.c_int64()
    _lib.check(_lib.lib().ql_gemm_mxfp4_workspace(*operand(a_shape), *operand(b_shape), ctypes.byref(size)))
    return size.value


def gemm_mxfp4(a: Float4Tensor, a_scales: torch.Tensor, b: Float4Tensor, b_scales: torch.Tensor, out_dtype: dt.dtype = dt.bfloat16,
               out=None) -> torch.Tensor:
    """dequantize_mxfp4(a) @ dequantize_mxfp4(b)^T on the block-scaled tensor cores: a [M, K] (activations, any M from one
    token up), b [N, K] (weights) and their scales as quantize_mxfp4 returns them; f32 sums, one rounding to `out_dtype`
    (float32, float16 or bfloat16)."""
    require_cuda(a, "a")
    require_cuda(b, "b")
    if not isinstance(a, Float4Tensor) or not isinstance(b, Float4Tensor):
        raise QuantizeError("gemm_mxfp4: a and b must be Float4Tensor, as quantize_mxfp4 returns them")
    if out is None and out_dtype not in dt.QUANTIZABLE_DTYPES:
        raise QuantizeError(f"Unsupported data type in gemm_mxfp4. Supported data types are: {dt.QUANTIZABLE_DTYPES}. Got out_dtype={out_dtype}")
    if len(a.shape) != 2 or len(b.shape) != 2 or a_scales.dim() != 2 or b_scales.dim() != 2:
        raise QuantizeError("gemm_mxfp4: data and scales must be 2-D")
    device = a.packed.device
    # dense, on a multiple of 4 bytes (a slice of rows need not be); kept alive across the call: a view only borrows the pointer
    sa, sb = a_scales.contiguous(), b_scales.contiguous()
    where = sa.data_ptr() | sb.data_ptr()
    if where % 4:
        sa, sb = sa.clone(), sb.clone()
        where = sa.data_ptr() | sb.data_ptr()
    other, y = (b, sa, sb), out
    if out is None:
        y = empty((a.shape[0], b.shape[0]), out_dtype.torch, device)
    else:
        other += (out,)
    ws, size = None, 0
    if where % 16 or a.shape[1] % 512:   # scale rows the kernel for many tokens wants a padded copy of
        size = _padding_bytes(a.shape, b.shape)
        if size:
            ws = empty((size,), torch.uint8, device)
    call_on(device, _lib.lib().ql_gemm_mxfp4, ql_view(a), ql_view(sa), ql_view(b), ql_view(sb), ql_view(y), ws.data_ptr() if size else None, size, same_device=other)
    return y
