"""Gated projection of a feed-forward block in 16 bits, and its backward pass: the unquantized counterpart of the fp8 block's
gate/up projection (mlp.gemm_fp8_swiglu), for the block that a quantized one is made from, compared with or trained as.  The
reference has no such operator; its pieces are tp.Linear and the activations of its frontend.

As all of the package, both functions work on plain tensors and record nothing for automatic differentiation: their results require
no gradient, whatever the operands do, and a training step calls gated_linear_backward itself."""
from __future__ import annotations

import ctypes
import functools

import torch

from . import _lib
from .ops import QuantizeError
from .tensor import call_on, empty, ql_view, require_cuda


def _activation(name: str) -> int:
    try:
        return _lib.ACTIVATIONS[name]
    except (KeyError, TypeError):
        raise QuantizeError(f"Unknown activation {name!r}: one of {tuple(_lib.ACTIVATIONS)}.") from None


def _rows(t: torch.Tensor, what: str) -> torch.Tensor:
    require_cuda(t, what)
    if t.dim() == 2:
        return t.contiguous()
    if t.dim() == 0:
        raise QuantizeError(f"{what} must have at least 1 dimension.")
    return t.reshape(-1, t.shape[-1]).contiguous() if t.numel() else t.reshape(t.shape[:-1].numel(), t.shape[-1])


@functools.lru_cache(maxsize=256)
def _workspace_bytes(x_shape, w_shape, dtype: int, want_dx: bool, want_dw: bool, device_index: int) -> int:
    """ql_gated_linear_backward_workspace, asked once per shape (and device, which is the current one)."""
    size = ctypes.c_int64()
    _lib.check(_lib.lib().ql_gated_linear_backward_workspace(_lib.make_tensor(None, dtype, x_shape), _lib.make_tensor(None, dtype, w_shape), want_dx, want_dw,
                                                             ctypes.byref(size)))
    return size.value


def gated_linear(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, activation: str = "silu", *, out=None) -> torch.Tensor:
    """act(x @ w_gate^T) * (x @ w_up^T): x [..., K], w_gate and w_up [I, K], all float16 or all bfloat16; both products,
    `activation` ("silu", "gelu", "gelu_tanh" or "relu") and the gate's product in one kernel, f32 sums, one rounding.  K and
    I are multiples of 8; any number of rows from none up.  The result is detached from operands that require gradients:
    gated_linear_backward gives theirs."""
    act = _activation(activation)
    x2 = _rows(x, "x")
    wg, wu = w_gate.contiguous(), w_up.contiguous()   # kept alive across the call: a view only borrows the pointer
    rows, I = x2.shape[0], wg.shape[0] if wg.dim() else 0   # what is no matrix the entry refuses
    if out is None:
        h = empty((rows, I), x.dtype, x.device)
    else:
        if tuple(out.shape) != tuple(x.shape[:-1]) + (I,):
            raise QuantizeError(f"out must have shape {tuple(x.shape[:-1]) + (I,)}, got {tuple(out.shape)}.")
        if not out.is_contiguous():
            raise QuantizeError("out must be contiguous (dense row-major).")
        h = out.view(rows, I)
    call_on(x.device, _lib.lib().ql_gated_linear, ql_view(x2), ql_view(wg), ql_view(wu), act, ql_view(h), same_device=(wg, wu, h))
    return out if out is not None else (h if x.dim() == 2 else h.view(x.shape[:-1] + (I,)))


def gated_linear_backward(grad: torch.Tensor, x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, activation: str = "silu", *,
                          need_input_grad: bool = True, need_weight_grad: bool = True):
    """(dx, dw_gate, dw_up) of gated_linear from `grad`, the gradient of its result [..., I]; None for what is not needed.
    Nothing is kept from the forward pass: the projections are computed again, their gradients are formed in f32 and rounded
    to the operands' type for the second products (of up to 64 tokens with the rounding's remainder beside it, so that only
    the results' own rounding is left).  In float16 they are held times a power of two chosen on the device from their largest
    magnitude: gradients may be of any size, and a token's keep all their digits down to 2^-16 of the largest.  Gradients have
    the type of what they belong to."""
    act = _activation(activation)
    x2, g2 = _rows(x, "x"), _rows(grad, "grad")
    if grad.shape[:-1] != x.shape[:-1]:
        raise QuantizeError(f"grad and x must have the same leading dimensions, got {tuple(grad.shape)} and {tuple(x.shape)}.")
    wg, wu = w_gate.contiguous(), w_up.contiguous()
    dtype, device = x.dtype, x.device
    dx = empty(x2.shape, dtype, device) if need_input_grad else None
    dwg = empty(wg.shape, dtype, device) if need_weight_grad else None
    dwu = empty(wu.shape, dtype, device) if need_weight_grad else None
    vx, vg = ql_view(x2), ql_view(wg)
    out = [ql_view(t) if t is not None else None for t in (dx, dwg, dwu)]
    L = _lib.lib()

    def run(stream):   # with the tensors' device current: the plan behind the workspace's size depends on the device
        size = _workspace_bytes(x2.shape, wg.shape, vx.dtype, need_input_grad, need_weight_grad, device.index)
        ws = empty((size,), torch.uint8, device)
        return L.ql_gated_linear_backward(ql_view(g2), vx, vg, ql_view(wu), act, *out, ws.data_ptr() or None, size, stream)
    call_on(device, run, same_device=(g2, wg, wu))
    return (dx.view(x.shape) if dx is not None and x.dim() != 2 else dx), dwg, dwu
