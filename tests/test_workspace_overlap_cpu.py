"""A workspace that shares memory with an operand or a result is refused.  Addresses only: nothing is launched."""
import ctypes

import pytest

from qlinear import _lib

B, F16 = _lib.BF16, _lib.F16


def _t(dtype, shape, ptr):
    return _lib.make_tensor(ptr, dtype, shape)


def _err(rc):
    assert rc == _lib.ERR_INVALID_ARGUMENT
    return _lib.lib().ql_last_error().decode()


def test_product():
    L = _lib.lib()
    M, N, K = 40, 72, 96   # rows of three scale bytes: more than 32 tokens need a padded copy of them
    at = {"a": 0x10000, "sa": 0x20000, "b": 0x30000, "sb": 0x40000, "y": 0x50000}
    t = [_t(_lib.F4E2M1, [M, K], at["a"]), _t(_lib.F8E8M0, [M, 3], at["sa"]), _t(_lib.F4E2M1, [N, K], at["b"]), _t(_lib.F8E8M0, [N, 3], at["sb"])]
    y = _t(_lib.F32, [M, N], at["y"])
    n = ctypes.c_int64()
    assert L.ql_gemm_mxfp4_workspace(*t, ctypes.byref(n)) == 0 and n.value > 0
    for ptr in list(at.values()) + [p + 16 for p in at.values()] + [p - n.value + 16 for p in at.values()]:
        assert "the workspace must not overlap" in _err(L.ql_gemm_mxfp4(*t, y, ptr // 16 * 16, n.value, None))


@pytest.mark.parametrize("dtype", [B, F16])
def test_gated_backward(dtype):
    L = _lib.lib()
    M, I, K = 512, 64, 128
    at = {"dh": 0x1000000, "x": 0x2000000, "wg": 0x3000000, "wu": 0x4000000, "dx": 0x5000000, "dwg": 0x6000000, "dwu": 0x7000000}
    shape = {"dh": [M, I], "x": [M, K], "wg": [I, K], "wu": [I, K], "dx": [M, K], "dwg": [I, K], "dwu": [I, K]}
    t = {k: _t(dtype, shape[k], at[k]) for k in at}
    n = ctypes.c_int64()
    assert L.ql_gated_linear_backward_workspace(t["x"], t["wg"], 1, 1, ctypes.byref(n)) == 0 and n.value > 0

    def call(ws):
        return L.ql_gated_linear_backward(t["dh"], t["x"], t["wg"], t["wu"], 0, t["dx"], t["dwg"], t["dwu"], ws, n.value, None)
    for ptr in list(at.values()) + [p + 256 for p in at.values()] + [(p - n.value + 256) // 256 * 256 for p in at.values()]:
        assert "the workspace must not overlap" in _err(call(ptr))
