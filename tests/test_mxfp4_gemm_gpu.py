"""The MXFP4 product against the product in float64 of the very same operands.

Bound: products of two e2m1 values under power-of-two scales are exact; an MMA adds 64 of them to the f32 accumulator and
may truncate where it aligns them, at most 2 steps of 2^-23 of the largest magnitude in the sum, which S = sum |a||b|
bounds.  With K / 64 MMAs and up to 8 partial sums added at the end, |error| <= (K / 64 + 8) 2^-22 S; the result type's
rounding, half a step (eps / 2 of the value, or half the smallest subnormal), comes on top."""
import numpy as np
import pytest
import torch

import mx_reference as mx
import qlinear as ql
from helpers import randn

pytestmark = pytest.mark.gpu


def operand(rows, K, seed, std=1.0):
    x = randn((rows, K), torch.float32, seed, std) * torch.exp(0.7 * randn((K,), torch.float32, seed + 1))
    return ql.quantize_mxfp4(x)


def wide(data, scales):
    codes = mx.unpack(data.packed.cpu().numpy(), data.shape)
    return torch.from_numpy(mx.values(codes, scales.view(torch.uint8).cpu().numpy())).cuda()


def check(y, a, sa, b, sb, K):
    A, B = wide(a, sa), wide(b, sb)
    want, S = A @ B.T, A.abs() @ B.abs().T
    f = torch.finfo(y.dtype)
    bound = (K / 64 + 8) * 2.0 ** -22 * S
    if y.dtype != torch.float32:
        bound = bound + f.eps / 2 * want.abs() + f.smallest_normal * f.eps / 2
    bad = ~((y.double() - want).abs() <= bound)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {float((y.double() - want).abs().max())}, first {bad.nonzero()[0].tolist()}"
    assert ql.lib().ql_gemm_status(None) == 0


def guarded(M, N, dtype):
    """A result with NaN rows before and behind it, to see what is written."""
    whole = torch.full((M + 2, N), float("nan"), dtype=dtype, device="cuda")
    return whole, whole[1:M + 1]


# rows, columns and K with tails; one token; K of one block, of less and more than a 256-value step; scale rows of every alignment
SMALL = [(1, 128, 256), (1, 1, 32), (3, 200, 96), (16, 129, 512), (17, 64, 2048), (32, 1000, 4128), (33, 130, 288), (64, 127, 1024), (65, 300, 320),
         (128, 128, 8192), (129, 500, 1056), (333, 1001, 2080), (5, 4096, 11008), (300, 40, 64)]


@pytest.mark.parametrize("M,N,K", SMALL)
@pytest.mark.parametrize("out", [torch.float32, torch.float16, torch.bfloat16])
def test_few_tiles(M, N, K, out):
    a, sa = operand(M, K, 5000 + M)
    b, sb = operand(N, K, 6000 + N, K ** -0.5)
    whole, y = guarded(M, N, out)
    ql.gemm_mxfp4(a, sa, b, sb, out=y)
    check(y, a, sa, b, sb, K)
    assert torch.isnan(whole[0]).all() and torch.isnan(whole[-1]).all()
    again = ql.gemm_mxfp4(a, sa, b, sb, out_dtype=ql.dtypes.from_torch(out))
    assert torch.equal(again, y)   # the same bits on every run


# many tiles: scales of whole 16-byte rows and padded ones, rows of Y of whole 16-byte pieces and of odd lengths
@pytest.mark.parametrize("M,N,K", [(2048, 4096, 512), (1700, 2600, 1056), (4100, 1120, 32), (2048, 2300, 2048), (640, 6700, 4640), (1701, 2601, 1280), (2047, 2305, 11008), (130, 4099, 544), (257, 2001, 1024), (2048, 1000, 4096), (70, 9000, 4096),
                                   (128, 11000, 8192), (3000, 101, 8192), (33, 9001, 4128), (40000, 101, 1024), (20000, 3, 4096),
                                   (512, 4096, 4096), (1024, 545, 2112), (500, 304, 8192), (130, 7777, 96)])
@pytest.mark.parametrize("out", [torch.float32, torch.float16, torch.bfloat16])
def test_many_tiles(M, N, K, out):
    a, sa = operand(M, K, 5100 + M)
    b, sb = operand(N, K, 6100 + N, K ** -0.5)
    whole, y = guarded(M, N, out)
    ql.gemm_mxfp4(a, sa, b, sb, out=y)
    check(y, a, sa, b, sb, K)
    assert torch.isnan(whole[0]).all() and torch.isnan(whole[-1]).all()


@pytest.mark.parametrize("M,N,K", [(2, 200, 288), (600, 9000, 288)])
def test_scales_of_every_size_and_nan(M, N, K):
    """Scales from 2^-100 to 2^100 that cancel in the product; a NaN scale spoils its own row or column only."""
    a, sa = operand(M, K, 5200)
    b, sb = operand(N, K, 6200)
    g = torch.Generator().manual_seed(7)
    e = torch.randint(-100, 101, (K // 32,), generator=g)
    sa8 = (sa.view(torch.uint8).int() + e.cuda()).to(torch.uint8).view(torch.float8_e8m0fnu)
    sb8 = (sb.view(torch.uint8).int() - e.cuda()).to(torch.uint8).view(torch.float8_e8m0fnu)
    y = ql.gemm_mxfp4(a, sa8, b, sb8, out_dtype=ql.float32)
    check(y, a, sa8, b, sb8, K)
    assert torch.equal(y, ql.gemm_mxfp4(a, sa, b, sb, out_dtype=ql.float32))
    sa8.view(torch.uint8)[1, 3] = 255
    sb8.view(torch.uint8)[7, 0] = 255
    z = ql.gemm_mxfp4(a, sa8, b, sb8, out_dtype=ql.float32)
    spoiled = torch.zeros_like(z, dtype=torch.bool)
    spoiled[1], spoiled[:, 7] = True, True
    assert torch.equal(torch.isnan(z), spoiled) and torch.equal(z[~spoiled], y[~spoiled])


@pytest.mark.parametrize("M,N", [(3, 70), (700, 9000)])
def test_sliced_operands(M, N):
    """Row slices: data start on whole rows of 16 bytes, scale rows of 33 and 5 bytes anywhere (a copy is made of those)."""
    for K in (1056, 160):
        a, sa = operand(M + 5, K, 5250)
        b, sb = operand(N + 5, K, 6250, K ** -0.5)
        part = lambda t, lo, n: ql.Float4Tensor(t.packed[lo * K // 2:(lo + n) * K // 2], (n, K))
        for lo in (1, 2, 4):
            a2, sa2, b2, sb2 = part(a, lo, M), sa[lo:lo + M], part(b, lo, N), sb[lo:lo + N]
            check(ql.gemm_mxfp4(a2, sa2, b2, sb2, out_dtype=ql.float32), a2, sa2, b2, sb2, K)


def test_streams_capture_and_interleaved_calls():
    """Calls on two streams at once, and two captured graphs replayed in turn, do not disturb one another."""
    cases = [(1, 4096, 8192), (700, 6000, 1056)]
    ops = [(operand(M, K, 5300 + i), operand(N, K, 6300 + i, K ** -0.5)) for i, (M, N, K) in enumerate(cases)]
    call = lambda i: ql.gemm_mxfp4(*ops[i][0], *ops[i][1])
    want = [call(0), call(1)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    torch.cuda.synchronize()
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(call(i))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i]) for i in range(2) for y in got[i])
    graphs, outs = [], []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call(i))
        graphs.append(g)
    for _ in range(3):
        for y in outs:
            y.fill_(float("nan"))
        for i, g in enumerate(graphs):
            with torch.cuda.stream(streams[i]):
                streams[i].wait_stream(torch.cuda.default_stream())
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(outs[i], want[i]) for i in range(2))
    assert ql.lib().ql_gemm_status(None) == 0


@pytest.mark.parametrize("N", [32768, 32771])
def test_offsets_beyond_32_bits(N):
    """Y of more than 2^31 values, rows of whole 16-byte pieces and odd ones: its last rows are what the same rows alone give
    (the few rows go through the other kernel: products of one block are exact in f32 either way)."""
    M, K = 70000, 32
    if torch.cuda.mem_get_info()[0] < 12 << 30:
        pytest.skip("needs 12 GB")
    a, sa = operand(M, K, 5500)
    b, sb = operand(N, K, 6500)
    y = ql.gemm_mxfp4(a, sa, b, sb)
    tail = ql.Float4Tensor(a.packed[-20 * K // 2:], (20, K))
    assert torch.equal(y[-20:], ql.gemm_mxfp4(tail, sa[-20:], b, sb))
    assert torch.equal(y[40000:40020], ql.gemm_mxfp4(ql.Float4Tensor(a.packed[40000 * K // 2:40020 * K // 2], (20, K)), sa[40000:40020], b, sb))


def test_calls_from_several_threads():
    """Host threads share nothing but caches: each on its own stream, few rows and many."""
    import threading
    shapes = [(1, 500, 1056), (40, 3000, 512), (300, 5000, 288), (300, 5001, 288)]
    ops = [(operand(M, K, 5600 + i), operand(N, K, 6600 + i, K ** -0.5)) for i, (M, N, K) in enumerate(shapes)]
    want = [ql.gemm_mxfp4(*a, *b) for a, b in ops]
    torch.cuda.synchronize()
    wrong = []

    def work(seed):
        with torch.cuda.stream(torch.cuda.Stream()):
            for k in range(12):
                i = (seed + k) % len(ops)
                y = ql.gemm_mxfp4(*ops[i][0], *ops[i][1])
                torch.cuda.current_stream().synchronize()
                if not torch.equal(y, want[i]):
                    wrong.append(i)
    threads = [threading.Thread(target=work, args=(s,)) for s in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_empty_and_refused():
    a, sa = operand(4, 64, 5400)
    b, sb = operand(8, 64, 6400)
    none = ql.quantize_mxfp4(torch.empty((0, 64), device="cuda"))
    assert ql.gemm_mxfp4(*none, b, sb).shape == (0, 8) and ql.gemm_mxfp4(a, sa, *none).shape == (4, 0)
    with pytest.raises(ql.QuantizeError, match="Float4Tensor"):
        ql.gemm_mxfp4(torch.ones((4, 64), device="cuda"), sa, b, sb)
    with pytest.raises(ql.QuantizeError, match="Unsupported data type"):
        ql.gemm_mxfp4(a, sa, b, sb, out_dtype=ql.int8)
    with pytest.raises(ql.QlError, match="one entry per block of 32"):
        ql.gemm_mxfp4(a, sb, b, sb)
    with pytest.raises(ql.QlError, match=r"y must be \[M,N\]"):
        ql.gemm_mxfp4(a, sa, b, sb, out=torch.empty((8, 4), device="cuda"))
    with pytest.raises(ql.QlError, match="one device"):
        ql.gemm_mxfp4(a, sa, b, sb, out=torch.empty((4, 8)))
    c, sc = ql.dynamic_quantize(torch.ones((8, 64), device="cuda"))   # NVFP4 scales are no MXFP4 scales
    with pytest.raises(ql.QlError, match="f8E8M0FNU"):
        ql.gemm_mxfp4(a, sa, c, sc)
