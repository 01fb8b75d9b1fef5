"""MXFP4 without a GPU: the host restatement on hand-worked blocks, and what the entry points refuse before they touch
a device."""
import ctypes

import numpy as np
import pytest
import torch

import mx_reference as mx
import qlinear as ql
from qlinear import _lib


def _t(dtype, shape, ptr=0x1000):
    return _lib.make_tensor(ptr, dtype, shape)


def _err(rc):
    assert rc != 0
    return _lib.lib().ql_last_error().decode()


def test_restatement_on_worked_blocks():
    x = np.zeros((7, 32))
    x[1, :8] = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 4.0]     # largest 5: scale 1, every tie to the even code
    x[2, 0], x[2, 1] = 7.99, -0.2                                # scale 1, saturates at 6; the small one rounds to -0
    x[3, 0] = 8.0                                                # the next binade: scale 2
    x[4, 0] = 2.0 ** -140                                        # below the smallest scale times the smallest step
    x[5, 0] = 3 * 2.0 ** -128                                    # smallest scale, code of 1.5
    x[6, 3] = np.inf
    codes, s = mx.quantize(x)
    assert s.ravel().tolist() == [0, 127, 127, 128, 0, 0, 255]
    assert codes[1, :8].tolist() == [0, 2, 2, 4, 4, 6, 6, 6]
    assert codes[2, :2].tolist() == [7, 8] and codes[3, 0] == 6 and codes[4, 0] == 0 and codes[5, 0] == 3
    assert np.isnan(mx.values(codes, s)[6]).all() and (codes[6] == 0).all()
    assert np.array_equal(mx.unpack(mx.pack(codes), codes.shape), codes)


def test_python_layer_refuses():
    with pytest.raises(ql.QlError, match="must live in GPU memory"):
        ql.quantize_mxfp4(torch.ones(4, 32))
    f4 = ql.Float4Tensor(torch.zeros(64, dtype=torch.uint8), (4, 32))
    with pytest.raises(ql.QlError, match="must live in GPU memory"):
        ql.dequantize_mxfp4(f4, torch.ones(4, 1).to(torch.float8_e8m0fnu))


def test_quantize_and_dequantize_argument_rules():
    L = _lib.lib()
    for fn, order in ((L.ql_quantize_mxfp4, lambda x, q, s: (x, q, s)), (L.ql_dequantize_mxfp4, lambda x, q, s: (q, s, x))):
        call = lambda x, q, s: fn(*order(x, q, s), None)
        x, q, s = _t(_lib.F32, [4, 64]), _t(_lib.F4E2M1, [4, 64]), _t(_lib.F8E8M0, [4, 2])
        assert "null tensor" in _err(call(x, q, None))
        assert "must be f32, f16 or bf16" in _err(call(_t(_lib.I8, [4, 64]), q, s))
        assert "data must be f4E2M1FN" in _err(call(x, _t(_lib.I4, [4, 64]), s))
        assert "scales f8E8M0FNU" in _err(call(x, q, _t(_lib.F8E4M3, [4, 2])))
        assert "same rank" in _err(call(x, q, _t(_lib.F8E8M0, [8])))
        assert "same rank" in _err(call(_t(_lib.F32, []), _t(_lib.F4E2M1, []), _t(_lib.F8E8M0, [])))
        assert "differ in shape" in _err(call(x, _t(_lib.F4E2M1, [4, 32]), s))
        assert "divisible by 32" in _err(call(_t(_lib.F32, [4, 48]), _t(_lib.F4E2M1, [4, 48]), _t(_lib.F8E8M0, [4, 1])))
        assert "one entry per block of 32" in _err(call(x, q, _t(_lib.F8E8M0, [4, 4])))
        assert "without data" in _err(call(x, _t(_lib.F4E2M1, [4, 64], None), s))
        assert "aligned" in _err(call(_t(_lib.F32, [4, 64], 0x1008), q, s))
        assert "aligned" in _err(call(x, _t(_lib.F4E2M1, [4, 64], 0x1002), s))
        assert call(_t(_lib.F32, [0, 64], None), _t(_lib.F4E2M1, [0, 64], None), _t(_lib.F8E8M0, [0, 2], None)) == 0


def test_product_argument_rules():
    L = _lib.lib()
    a, sa, b, sb, y = _t(_lib.F4E2M1, [4, 64]), _t(_lib.F8E8M0, [4, 2]), _t(_lib.F4E2M1, [8, 64]), _t(_lib.F8E8M0, [8, 2]), _t(_lib.BF16, [4, 8])
    call = lambda a=a, sa=sa, b=b, sb=sb, y=y, ws=None, n=0: L.ql_gemm_mxfp4(a, sa, b, sb, y, ws, n, None)
    assert "a is null" in _err(call(sa=None)) and "b is null" in _err(call(b=None))
    assert "data must be f4E2M1FN" in _err(call(a=_t(_lib.I4, [4, 64])))
    assert "scales f8E8M0FNU" in _err(call(sb=_t(_lib.F8E4M3, [8, 2])))
    assert "must be 2-D" in _err(call(a=_t(_lib.F4E2M1, [256])))
    assert "one entry per block of 32" in _err(call(sa=_t(_lib.F8E8M0, [4, 4])))
    assert "one entry per block of 32" in _err(call(a=_t(_lib.F4E2M1, [4, 48]), sa=_t(_lib.F8E8M0, [4, 1])))
    assert "inner dimensions differ" in _err(call(b=_t(_lib.F4E2M1, [8, 32]), sb=_t(_lib.F8E8M0, [8, 1])))
    assert "y must be [M,N]" in _err(call(y=_t(_lib.BF16, [8, 4])))
    assert "f32, f16 or bf16" in _err(call(y=_t(_lib.I8, [4, 8])))
    assert "no data pointer" in _err(call(y=_t(_lib.BF16, [4, 8], None)))
    assert "non-zero K" in _err(call(a=_t(_lib.F4E2M1, [4, 0], None), sa=_t(_lib.F8E8M0, [4, 0], None), b=_t(_lib.F4E2M1, [8, 0], None), sb=_t(_lib.F8E8M0, [8, 0], None)))
    assert "16-byte aligned" in _err(call(b=_t(_lib.F4E2M1, [8, 64], 0x1008)))
    assert "4-byte aligned scales" in _err(call(sb=_t(_lib.F8E8M0, [8, 2], 0x1002)))
    assert "aligned to its type" in _err(call(y=_t(_lib.BF16, [4, 8], 0x1001)))
    assert call(a=_t(_lib.F4E2M1, [0, 64], None), sa=_t(_lib.F8E8M0, [0, 2], None), y=_t(_lib.BF16, [0, 8], None)) == 0
    # many tokens whose scale rows are no multiple of 16 bytes: a workspace for a padded copy
    size = ctypes.c_int64(-1)
    many = dict(a=_t(_lib.F4E2M1, [40, 96]), sa=_t(_lib.F8E8M0, [40, 3]), b=_t(_lib.F4E2M1, [8, 96]), sb=_t(_lib.F8E8M0, [8, 3]))
    assert L.ql_gemm_mxfp4_workspace(*many.values(), ctypes.byref(size)) == 0 and size.value == 48 * 16
    y = _t(_lib.BF16, [40, 8])
    assert "needs a workspace of 768 bytes" in _err(call(**many, y=y)) and "needs a workspace of 768 bytes" in _err(call(**many, y=y, ws=0x1000, n=767))
    assert "16-byte aligned" in _err(call(**many, y=y, ws=0x1008, n=768))
    assert L.ql_gemm_mxfp4_workspace(a, sa, b, sb, ctypes.byref(size)) == 0 and size.value == 0
    assert "no place for the size" in _err(L.ql_gemm_mxfp4_workspace(a, sa, b, sb, None))


def test_results_that_share_memory_are_refused():
    """Addresses only: the refusals come before anything is launched."""
    L = _lib.lib()
    x, q, s = _t(_lib.F32, [4, 64], 0x10000), _t(_lib.F4E2M1, [4, 64], 0x20000), _t(_lib.F8E8M0, [4, 2], 0x30000)
    assert "must not overlap" in _err(L.ql_quantize_mxfp4(x, _t(_lib.F4E2M1, [4, 64], 0x10000), s, None))
    assert "must not overlap" in _err(L.ql_quantize_mxfp4(x, q, _t(_lib.F8E8M0, [4, 2], 0x10000 + 1023), None))
    assert "must not overlap" in _err(L.ql_quantize_mxfp4(x, q, _t(_lib.F8E8M0, [4, 2], 0x20000 + 127), None))
    assert "must not overlap" in _err(L.ql_dequantize_mxfp4(q, s, _t(_lib.F32, [4, 64], 0x20000 - 512), None))
    assert "must not overlap" in _err(L.ql_dequantize_mxfp4(q, s, _t(_lib.BF16, [4, 64], 0x30000), None))
    b, sb = _t(_lib.F4E2M1, [8, 64], 0x40000), _t(_lib.F8E8M0, [8, 2], 0x50000)
    for ptr in (0x20000, 0x30000, 0x40000 + 256 - 2, 0x50000 - 62):
        assert "must not overlap" in _err(L.ql_gemm_mxfp4(q, s, b, sb, _t(_lib.BF16, [4, 8], ptr), None, 0, None))


def test_python_layer_refuses_scales_of_other_ranks():
    class OnGpu(ql.Float4Tensor):   # passes for one in GPU memory; the refusal comes before anything is read
        device = torch.device("cuda", 0)
    a = OnGpu(torch.zeros(64, dtype=torch.uint8), (4, 32))
    s = torch.zeros(4, 1, dtype=torch.uint8).view(torch.float8_e8m0fnu)
    for bad in ((a, s.view(4), a, s), (a, s, a, s[0, 0])):
        with pytest.raises(ql.QuantizeError, match="must be 2-D"):
            ql.gemm_mxfp4(*bad)
