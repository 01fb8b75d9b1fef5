"""MXFP4 kernels against the host restatement in float64 (mx_reference): data and scales bit for bit, values bit for bit."""
import numpy as np
import pytest
import torch

import mx_reference as mx
import qlinear as ql
from helpers import randn

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]


def bits(t):
    return t.contiguous().view(torch.uint8).cpu().numpy()


def check_quantized(x):
    data, scales = ql.quantize_mxfp4(x)
    assert data.shape == tuple(x.shape) and scales.dtype == torch.float8_e8m0fnu and tuple(scales.shape) == tuple(x.shape[:-1]) + (x.shape[-1] // 32,)
    codes, s = mx.quantize(x.double().cpu().numpy())
    assert np.array_equal(bits(scales).reshape(s.shape), s)
    assert np.array_equal(data.packed.cpu().numpy(), mx.pack(codes))
    return data, scales, codes, s


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1, 32), (7, 96), (32,), (3, 5, 160), (1, 8192), (1021, 416), (0, 64), (4, 0), (2, 3, 1, 64)])
def test_round_trip(dtype, shape):
    x = randn(shape, dtype, 4000 + sum(shape), std=3.0) * torch.exp(2 * randn(shape[-1:], torch.float32, 4001)).to(dtype)
    if x.numel() == 0:
        data, scales = ql.quantize_mxfp4(x)
        assert ql.dequantize_mxfp4(data, scales).shape == x.shape
        return
    data, scales, codes, s = check_quantized(x)
    want = torch.from_numpy(mx.values(codes, s))
    for out in (ql.float32, ql.float16, ql.bfloat16):   # float64 -> float32 is exact here, so this rounds once
        assert torch.equal(ql.dequantize_mxfp4(data, scales, out).cpu(), want.float().to(out.torch))


@pytest.mark.parametrize("dtype", TYPES)
def test_every_16_bit_pattern_and_binade(dtype):
    """Blocks whose first value runs through every 16-bit pattern (for f32: the patterns as upper halves), the rest
    spread below it: ties, subnormals, infinities and NaN of every binade."""
    p = torch.arange(65536, dtype=torch.int32)
    lead = p.to(torch.int16).view(dtype) if dtype != torch.float32 else (p << 16).view(torch.float32)
    # 1, 7/8, ... of the largest: multiples of 1/8 of a power of two fall on e2m1's ties
    f = torch.cat([torch.tensor([1.0]), torch.arange(1, 32) / 32.0 * torch.tensor([1.0, -1.0]).repeat(16)[:31]])
    x = (lead.double()[:, None] * f.double()).to(dtype)
    x[:, 0] = lead
    x = x.cuda()
    data, scales = ql.quantize_mxfp4(x)
    codes, s = mx.quantize(x.double().cpu().numpy())
    assert np.array_equal(bits(scales).reshape(s.shape), s)
    assert np.array_equal(data.packed.cpu().numpy(), mx.pack(codes))


def test_blocks_with_infinities_and_nan_stay_apart():
    x = randn((6, 96), torch.float32, 4010)
    x[0, 3], x[1, 40], x[2, 95], x[3, 32:64] = float("inf"), float("nan"), -float("inf"), 0.0
    x[4, 0] = -0.0
    data, scales, codes, s = check_quantized(x)
    y = ql.dequantize_mxfp4(data, scales)
    bad = torch.zeros(6, 3, dtype=torch.bool)
    bad[0, 0] = bad[1, 1] = bad[2, 2] = True
    assert torch.equal(torch.isnan(y).cpu(), bad.repeat_interleave(32, dim=1))
    assert (y[3, 32:64] == 0).all() and float(s[3, 1]) == 0
    assert torch.signbit(y[4, 0]).item()


@pytest.mark.parametrize("out", [ql.float32, ql.float16, ql.bfloat16])
def test_dequantize_takes_every_scale_and_code(out):
    codes = np.tile(np.arange(16, dtype=np.uint8), (256, 2))
    s = np.arange(256, dtype=np.uint8).reshape(256, 1)
    data = ql.Float4Tensor(torch.from_numpy(mx.pack(codes)).cuda(), (256, 32))
    y = ql.dequantize_mxfp4(data, torch.from_numpy(s).cuda().view(torch.float8_e8m0fnu), out)
    want = torch.from_numpy(mx.values(codes, s)).float().to(out.torch)   # f32 overflows to infinity where the product does
    assert torch.equal(torch.isnan(y).cpu(), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(y.float().cpu(), nan=0.0, posinf=1e39, neginf=-1e39), torch.nan_to_num(want.float(), nan=0.0, posinf=1e39, neginf=-1e39))


def test_strided_input_another_stream_and_capture():
    base = randn((64, 512), torch.bfloat16, 4020)
    x = base.t()[:, :32].contiguous().t()          # a transposed, strided view goes through a dense copy
    check_quantized(base[:, 64:192])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        data, scales = ql.quantize_mxfp4(base)
        y = ql.dequantize_mxfp4(data, scales, ql.bfloat16)
    torch.cuda.current_stream().wait_stream(side)
    want = ql.dequantize_mxfp4(*ql.quantize_mxfp4(base), ql.bfloat16)
    assert torch.equal(y, want) and x.shape == (32, 512)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        d2, s2 = ql.quantize_mxfp4(base)
        y2 = ql.dequantize_mxfp4(d2, s2, ql.bfloat16)
    base.copy_(randn((64, 512), torch.bfloat16, 4021, std=5.0))
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(y2, ql.dequantize_mxfp4(*ql.quantize_mxfp4(base), ql.bfloat16)) and not torch.equal(y2, want)


def test_more_values_than_32_bits_count():
    """Over 2^31 values: the tail beyond every 32-bit offset is quantized and dequantized as the same rows alone are."""
    rows, cols = 65537 + 8, 32768
    if torch.cuda.mem_get_info()[0] < 16 << 30:
        pytest.skip("needs 16 GB")
    x = torch.zeros((rows, cols), dtype=torch.bfloat16, device="cuda")
    x[-8:] = randn((8, cols), torch.bfloat16, 4030)
    data, scales = ql.quantize_mxfp4(x)
    tail, ts = ql.quantize_mxfp4(x[-8:])
    assert torch.equal(data.packed[-8 * cols // 2:], tail.packed) and np.array_equal(bits(scales[-8:]), bits(ts))
    y = ql.dequantize_mxfp4(data, scales, ql.bfloat16)
    assert torch.equal(y[-8:], ql.dequantize_mxfp4(tail, ts, ql.bfloat16)) and not y[:8].any()


def test_refusals():
    with pytest.raises(ql.QuantizeError, match="divisible by 32"):
        ql.quantize_mxfp4(torch.ones((4, 48), device="cuda"))
    with pytest.raises(ql.QuantizeError, match="divisible by 32"):
        ql.quantize_mxfp4(torch.ones((), device="cuda"))
    with pytest.raises(ql.QuantizeError, match="valid dtype"):
        ql.quantize_mxfp4(torch.ones((4, 32), dtype=torch.int8, device="cuda"))
    data, scales = ql.quantize_mxfp4(torch.ones((4, 64), device="cuda"))
    with pytest.raises(ql.QuantizeError, match="Unsupported data type"):
        ql.dequantize_mxfp4(data, scales, ql.int8)
    with pytest.raises(ql.QlError, match="one entry per block of 32"):
        ql.dequantize_mxfp4(data, scales[:, :1])
    with pytest.raises(ql.QlError, match="f8E8M0FNU"):
        ql.dequantize_mxfp4(data, scales.float())
    with pytest.raises(ql.QlError, match="one device"):
        ql.dequantize_mxfp4(data, scales, out=torch.empty((4, 64)))
    with pytest.raises(ql.QlError, match="differ in shape"):
        ql.dequantize_mxfp4(data, scales, out=torch.empty((4, 32), device="cuda"))
    with pytest.raises(ql.QlError, match="aligned"):
        ql.quantize_mxfp4(torch.ones(4 * 64 + 1, device="cuda")[1:].view(4, 64))
