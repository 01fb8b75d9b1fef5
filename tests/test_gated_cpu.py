"""The gated projection without a GPU: what its entry points refuse before they touch a device."""
import ctypes

import pytest
import torch

import qlinear as ql
from qlinear import _lib


def _t(dtype, shape, ptr=0x1000):
    return _lib.make_tensor(ptr, dtype, shape)


def _err(rc):
    assert rc != 0
    return _lib.lib().ql_last_error().decode()


def test_python_layer_refuses():
    x, w = torch.ones(4, 16, dtype=torch.bfloat16), torch.ones(8, 16, dtype=torch.bfloat16)
    with pytest.raises(ql.QuantizeError, match="Unknown activation"):
        ql.gated_linear(x, w, w, "swish")
    with pytest.raises(ql.QlError, match="must live in GPU memory"):
        ql.gated_linear(x, w, w)
    with pytest.raises(ql.QuantizeError, match="Unknown activation"):
        ql.gated_linear_backward(torch.ones(4, 8), x, w, w, None)
    with pytest.raises(ql.QlError, match="must live in GPU memory"):
        ql.gated_linear_backward(torch.ones(4, 8), x, w, w)


B = _lib.BF16


def _common(call, h_name):
    assert "x is null" in _err(call(x=None)) and "w_up is null" in _err(call(wu=None))
    assert "must be a 2-D tensor" in _err(call(x=_t(B, [64])))
    assert "must be f16 or bf16" in _err(call(x=_t(_lib.F32, [4, 16])))
    assert "of one type" in _err(call(wu=_t(_lib.F16, [8, 16])))
    assert "must both be [I,K]" in _err(call(wg=_t(B, [8, 24])))
    assert "must both be [I,K]" in _err(call(wu=_t(B, [16, 16])))
    assert f"{h_name} must be [M,I]" in _err(call(h=_t(B, [4, 16])))
    assert "unknown activation" in _err(call(act=4)) and "unknown activation" in _err(call(act=-1))
    assert "no data pointer" in _err(call(wg=_t(B, [8, 16], None)))
    assert "16-byte aligned" in _err(call(wg=_t(B, [8, 16], 0x1002)))
    assert "multiples of 8" in _err(call(x=_t(B, [4, 12]), wg=_t(B, [8, 12]), wu=_t(B, [8, 12])))
    assert "multiples of 8" in _err(call(wg=_t(B, [12, 16]), wu=_t(B, [12, 16]), h=_t(B, [4, 12])))


def test_forward_argument_rules():
    L = _lib.lib()
    t = dict(x=_t(B, [4, 16]), wg=_t(B, [8, 16]), wu=_t(B, [8, 16]), h=_t(B, [4, 8]), act=0)

    def call(**kw):
        a = {**t, **kw}
        return L.ql_gated_linear(a["x"], a["wg"], a["wu"], a["act"], a["h"], None)
    _common(call, "h")
    assert call(x=_t(B, [0, 16], None), h=_t(B, [0, 8], None)) == 0


def test_backward_argument_rules():
    L = _lib.lib()
    t = dict(h=_t(B, [4, 8]), x=_t(B, [4, 16]), wg=_t(B, [8, 16]), wu=_t(B, [8, 16]), act=0, dx=_t(B, [4, 16]), dg=_t(B, [8, 16]), du=_t(B, [8, 16]), ws=None, n=0)

    def call(**kw):
        a = {**t, **kw}
        return L.ql_gated_linear_backward(a["h"], a["x"], a["wg"], a["wu"], a["act"], a["dx"], a["dg"], a["du"], a["ws"], a["n"], None)
    _common(call, "grad")
    assert "go together" in _err(call(dg=None))
    assert "dx must have the type and shape" in _err(call(dx=_t(B, [4, 24])))
    assert "dw_up must have the type and shape" in _err(call(du=_t(_lib.F16, [8, 16])))
    assert "dx must be 16-byte aligned" in _err(call(dx=_t(B, [4, 16], 0x1008)))
    assert "dw_gate has no data pointer" in _err(call(dg=_t(B, [8, 16], None)))
    assert "needs a workspace of" in _err(call())
    assert "needs a workspace of" in _err(call(ws=0x1000, n=16))
    n = ctypes.c_int64(-1)
    assert L.ql_gated_linear_backward_workspace(t["x"], t["wg"], 1, 1, ctypes.byref(n)) == 0 and n.value > 0
    assert "256-byte aligned" in _err(call(ws=0x1010, n=n.value))
    assert L.ql_gated_linear_backward_workspace(_t(B, [0, 16], None), t["wg"], 1, 1, ctypes.byref(n)) == 0 and n.value == 0
    assert "needs x" in _err(L.ql_gated_linear_backward_workspace(None, t["wg"], 1, 1, ctypes.byref(n)))
    assert call(dx=None, dg=None, du=None) == 0   # nothing asked for


def test_results_that_share_memory_are_refused():
    """Addresses only: the refusals come before anything is launched."""
    L = _lib.lib()
    x, wg, wu = _t(B, [4, 16], 0x10000), _t(B, [8, 16], 0x20000), _t(B, [8, 16], 0x30000)
    for ptr in (0x10000, 0x10000 + 4 * 16 * 2 - 16, 0x20000 - 16, 0x30000 + 8 * 16 * 2 - 16):
        assert "h must not overlap an operand" in _err(L.ql_gated_linear(x, wg, wu, 0, _t(B, [4, 8], ptr), None))
    n = ctypes.c_int64()
    assert L.ql_gated_linear_backward_workspace(x, wg, 1, 1, ctypes.byref(n)) == 0

    def call(dx=0x50000, dwg=0x60000, dwu=0x70000):
        return L.ql_gated_linear_backward(_t(B, [4, 8], 0x40000), x, wg, wu, 0, _t(B, [4, 16], dx), _t(B, [8, 16], dwg), _t(B, [8, 16], dwu), 0x100000, n.value, None)
    assert "dx must not overlap an operand" in _err(call(dx=0x10000))
    assert "dw_gate must not overlap an operand" in _err(call(dwg=0x40000))
    assert "dw_up must not overlap an operand" in _err(call(dwu=0x30000 - 16))
    assert "dw_gate and dw_up must not overlap" in _err(call(dwu=0x60000))
    assert "dx and dw_gate must not overlap" in _err(call(dx=0x60010))
