"""The gated projection and its gradients against the formulas in float64.

Bounds, worst case: an MMA adds 16 products to the f32 accumulator and may truncate where it aligns them, at most 2 steps of
2^-23 of the largest magnitude in the sum: e = (K / 16 + 8) 2^-22 sum |x||w| for a projection.  The activation and its slope use
the fast exponential and division, well within 2^-15 of values of order |z| and 1.  |act'| <= 1.2, |act''| <= 1 for the smooth
ones; a relu's slope is undecided where |g| <= e.  dG and dU are rounded to the operands' type (half a step, eps / 2) before the
second products, whose sums again lose 2^-22 of the sum of magnitudes per MMA; the result's rounding comes on top."""
import math

import pytest
import torch

import qlinear as ql
from helpers import randn

pytestmark = pytest.mark.gpu

ACTS = ["silu", "gelu", "gelu_tanh", "relu"]


def act_both(z, name):
    if name == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s))
    if name == "gelu":
        c = 0.5 * torch.erfc(-z / math.sqrt(2))
        return z * c, c + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if name == "gelu_tanh":
        k = math.sqrt(2 / math.pi)
        t = torch.tanh(k * (z + 0.044715 * z ** 3))
        return z * (1 + t) / 2, (1 + t) / 2 + z / 2 * (1 - t * t) * k * (1 + 3 * 0.044715 * z * z)
    return z.clamp(min=0), (z > 0).double()


class Case:
    def __init__(self, M, I, K, dtype, act, seed, scale=1.0):
        self.M, self.I, self.K, self.dtype, self.act = M, I, K, dtype, act
        self.x = randn((M, K), dtype, seed)
        self.wg = randn((I, K), dtype, seed + 1, scale * K ** -0.5)
        self.wu = randn((I, K), dtype, seed + 2, scale * K ** -0.5)
        self.dh = randn((M, I), dtype, seed + 3, 0.5)

    def exact(self):
        x, wg, wu, dh = (t.double() for t in (self.x, self.wg, self.wu, self.dh))
        f = torch.finfo(self.dtype)
        half, tiny = f.eps / 2, f.smallest_normal * f.eps / 2
        g, u = x @ wg.T, x @ wu.T
        a, d = act_both(g, self.act)
        k = (self.K / 16 + 8) * 2.0 ** -22
        eg, eu = k * (x.abs() @ wg.abs().T), k * (x.abs() @ wu.abs().T)
        ea = 1.2 * eg + 2.0 ** -15 * (a.abs() + 2.0 ** -10)
        eh = ea * u.abs() + a.abs() * eu + ea * eu
        h = a * u
        self.h, self.h_bound = h, eh + half * (h.abs() + eh) + tiny
        dg, du = dh * u * d, dh * a
        ed = eg + 2.0 ** -15 * (1 + g.abs()) if self.act != "relu" else (g.abs() <= eg).double()
        e_dg = dh.abs() * (u.abs() * ed + 1.2 * eu + ed * eu)
        e_du = dh.abs() * ea
        e_dg, e_du = e_dg + half * (dg.abs() + e_dg) + tiny, e_du + half * (du.abs() + e_du) + tiny
        n2, nm = (2 * self.I / 16 + 40) * 2.0 ** -22, (self.M / 16 + 40) * 2.0 ** -22
        fin = lambda want, e: (want, e + half * (want.abs() + e) + tiny)
        self.dx = fin(dg @ wg + du @ wu, (e_dg + n2 * dg.abs()) @ wg.abs() + (e_du + n2 * du.abs()) @ wu.abs())
        self.dwg = fin(dg.T @ x, (e_dg + nm * dg.abs()).T @ x.abs())
        self.dwu = fin(du.T @ x, (e_du + nm * du.abs()).T @ x.abs())
        return self


def close(got, want, bound, what):
    bad = ~((got.double() - want).abs() <= bound)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, first {bad.nonzero()[0].tolist()}, worst {float((got.double() - want).abs().nan_to_num(9e9).max())}"


def near(got, want, dtype, what):
    """Over all values the roundings average out: sqrt(2) of the result type's own rounding (eps / 2 / sqrt(3) of the value, at
    most), with a quarter to spare."""
    rel = float((got.double() - want).norm() / want.norm())
    assert rel <= 1.25 * math.sqrt(2) * torch.finfo(dtype).eps / 2 / math.sqrt(3), f"{what}: {rel}"


def guarded(rows, cols, dtype):
    whole = torch.full((rows + 2, cols), float("nan"), dtype=dtype, device="cuda")
    return whole, whole[1:rows + 1]


# rows: one, below, at and above a token tile, many; channels and K with tails of every kind; K below and above a step of 64
SMALL = [(1, 128, 64), (1, 8, 8), (2, 40, 72), (16, 1000, 520), (17, 264, 128), (33, 136, 1032), (64, 2744, 192), (65, 512, 320), (100, 72, 4096),
         (211, 2744, 1032), (1, 11008, 4096)]
LARGE = [(1100, 4104, 136), (2000, 2056, 520), (600, 8200, 72), (4097, 1032, 264)]


@pytest.mark.parametrize("M,I,K", SMALL + LARGE)
@pytest.mark.parametrize("dtype,act", [(torch.bfloat16, "silu"), (torch.float16, "gelu"), (torch.bfloat16, "gelu_tanh"), (torch.float16, "relu")])
def test_forward(M, I, K, dtype, act):
    c = Case(M, I, K, dtype, act, 7000 + M + I, scale=2.0).exact()
    whole, h = guarded(M, I, dtype)
    ql.gated_linear(c.x, c.wg, c.wu, act, out=h)
    assert ql.lib().ql_gemm_status(None) == 0
    close(h, c.h, c.h_bound, f"{M}x{I}x{K} {act}")
    assert torch.isnan(whole[0]).all() and torch.isnan(whole[-1]).all()
    assert torch.equal(ql.gated_linear(c.x, c.wg, c.wu, act), h)   # the same bits on every run


BACK = [(1, 128, 64), (1, 8, 8), (3, 40, 72), (77, 2744, 1032), (64, 264, 520), (130, 136, 264), (300, 1000, 328), (1, 4096, 1024), (2500, 72, 40),
        (700, 2056, 1544), (1030, 4104, 520)]


@pytest.mark.parametrize("M,I,K", BACK)
@pytest.mark.parametrize("dtype,act", [(torch.bfloat16, "silu"), (torch.float16, "gelu"), (torch.float16, "gelu_tanh"), (torch.bfloat16, "relu")])
def test_backward(M, I, K, dtype, act):
    c = Case(M, I, K, dtype, act, 7500 + M + I).exact()
    dx, dwg, dwu = ql.gated_linear_backward(c.dh, c.x, c.wg, c.wu, act)
    assert ql.lib().ql_gemm_status(None) == 0
    for got, (want, bound), what in ((dx, c.dx, "dx"), (dwg, c.dwg, "dw_gate"), (dwu, c.dwu, "dw_up")):
        assert got.dtype == dtype and got.shape == want.shape
        close(got, want, bound, f"{what} {M}x{I}x{K} {act}")
        if M * I >= 4096 and want.numel() >= 4096:
            near(got, want, dtype, what)
    again = ql.gated_linear_backward(c.dh, c.x, c.wg, c.wu, act)
    assert all(torch.equal(a, b) for a, b in zip((dx, dwg, dwu), again))
    only_x = ql.gated_linear_backward(c.dh, c.x, c.wg, c.wu, act, need_weight_grad=False)
    only_w = ql.gated_linear_backward(c.dh, c.x, c.wg, c.wu, act, need_input_grad=False)
    assert only_x[1] is None and only_x[2] is None and only_w[0] is None
    close(only_x[0], *c.dx, "dx alone")
    close(only_w[1], *c.dwg, "dw_gate alone")
    close(only_w[2], *c.dwu, "dw_up alone")


@pytest.mark.parametrize("act", ACTS)
def test_gradients_against_differences(act):
    """Differences of L = sum(h * dh) along random directions, with the formulas' h in float64 (the step's own error is of the
    order of step^2 for the smooth ones; a relu is left out where a step crosses its kink)."""
    M, I, K = 24, 96, 64
    c = Case(M, I, K, torch.float16, act, 7900).exact()
    grads = ql.gated_linear_backward(c.dh, c.x, c.wg, c.wu, act)
    leaves = [t.double() for t in (c.x, c.wg, c.wu)]
    step = 1e-6
    for i, (grad, (_, bound)) in enumerate(zip(grads, (c.dx, c.dwg, c.dwu))):
        v = randn(tuple(leaves[i].shape), torch.float64, 7910 + i)

        def loss(s):
            t = [leaf + s * v if j == i else leaf for j, leaf in enumerate(leaves)]
            return t[0] @ t[1].T, (act_both(t[0] @ t[1].T, act)[0] * (t[0] @ t[2].T) * c.dh.double())
        (g1, l1), (g0, l0) = loss(step), loss(-step)
        crossed = (g1 > 0) != (g0 > 0) if act == "relu" else torch.zeros_like(g1, dtype=torch.bool)
        assert not crossed.any()
        difference = float((l1 - l0).sum()) / (2 * step)
        slope = float((grad.double() * v).sum())
        assert abs(slope - difference) <= float((bound * v.abs()).sum()) + 1e-5 * float(((l1 - l0).abs() / (2 * step)).sum())


@pytest.mark.parametrize("act", ACTS)
def test_extreme_values(act):
    """Projections far out on both sides, zeros, an infinity and a NaN: H is what the formula gives, and rows do not mix."""
    K = I = 64
    x = torch.zeros((8, K), dtype=torch.bfloat16, device="cuda")
    x[0, 0], x[1, 0], x[2, 0], x[3, 0], x[5, 0], x[6, 0] = 200.0, -200.0, 3e4, -3e4, float("inf"), float("nan")
    eye = torch.eye(I, K, dtype=torch.bfloat16, device="cuda")
    h = ql.gated_linear(x[:5].contiguous(), eye, eye, act).double()
    want = act_both(x[:5].double(), act)[0] * x[:5].double()
    assert torch.allclose(h, want, rtol=2.0 ** -8, atol=1e-30)
    h = ql.gated_linear(x, eye, eye, act)
    assert torch.isnan(h[6]).any() and torch.equal(torch.isnan(h[:5]), torch.zeros_like(h[:5], dtype=torch.bool)) and not torch.isnan(h[7]).any()
    dx, dwg, dwu = ql.gated_linear_backward(torch.ones((4, I), dtype=torch.bfloat16, device="cuda"), x[:4].contiguous(), eye, eye, act)
    assert torch.isfinite(dx).all() and torch.isfinite(dwg).all() and torch.isfinite(dwu).all()


def test_leading_dimensions_strides_and_empty():
    c = Case(24, 72, 40, torch.bfloat16, "silu", 8000).exact()
    h = ql.gated_linear(c.x.view(2, 3, 4, 40), c.wg, c.wu)
    assert h.shape == (2, 3, 4, 72)
    close(h.reshape(24, 72), c.h, c.h_bound, "leading dimensions")
    assert ql.gated_linear(c.x[0], c.wg, c.wu).shape == (72,)
    wide = torch.cat([c.x, c.x], dim=1)
    assert torch.equal(ql.gated_linear(wide[:, 40:], c.wg, c.wu), h.reshape(24, 72))                       # a strided view
    assert torch.equal(ql.gated_linear(c.x, c.wg.t().contiguous().t(), c.wu), h.reshape(24, 72))           # a transposed weight
    dx, dwg, dwu = ql.gated_linear_backward(c.dh.view(2, 3, 4, 72), c.x.view(2, 3, 4, 40), c.wg, c.wu)
    assert dx.shape == (2, 3, 4, 40)
    close(dx.reshape(24, 40), *c.dx, "dx")
    one = c.dh[:1].expand(24, 72)                                                                           # a broadcast gradient
    got = ql.gated_linear_backward(one, c.x, c.wg, c.wu)
    want = ql.gated_linear_backward(one.contiguous(), c.x, c.wg, c.wu)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    none = c.x[:0]
    assert ql.gated_linear(none, c.wg, c.wu).shape == (0, 72)
    dx, dwg, dwu = ql.gated_linear_backward(c.dh[:0], none, c.wg, c.wu)
    assert dx.shape == (0, 40) and not dwg.any() and not dwu.any()
    dx, dwg, dwu = ql.gated_linear_backward(c.dh[:, :0], c.x, c.wg[:0], c.wu[:0])
    assert not dx.any() and dwg.shape == (0, 40)
    assert not ql.gated_linear(c.x[:, :0], c.wg[:, :0], c.wu[:, :0]).any()


def test_the_same_tensor_twice():
    c = Case(40, 64, 64, torch.float16, "gelu", 8100)
    c.wu = c.wg
    c.exact()
    close(ql.gated_linear(c.x, c.wg, c.wg, "gelu"), c.h, c.h_bound, "one weight for both")
    dx, dwg, dwu = ql.gated_linear_backward(c.dh, c.x, c.wg, c.wg, "gelu")
    close(dx, *c.dx, "dx")
    close(dwg, *c.dwg, "dw_gate")
    close(dwu, *c.dwu, "dw_up")


def test_streams_and_capture():
    """Forward and backward on two streams at once, and two captured graphs replayed in turn on them."""
    cases = [Case(5, 1032, 264, torch.bfloat16, "silu", 8200), Case(700, 2056, 520, torch.bfloat16, "gelu", 8210)]

    def step(c):
        return (ql.gated_linear(c.x, c.wg, c.wu, c.act),) + ql.gated_linear_backward(c.dh, c.x, c.wg, c.wu, c.act)
    want = [step(c) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(4):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(step(cases[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for i in range(2) for r in got[i] for a, b in zip(r, want[i]))
    graphs, outs = [], []
    for c in cases:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(c))
        graphs.append(g)
    for _ in range(3):
        for r in outs:
            for t in r:
                t.fill_(float("nan"))
        torch.cuda.synchronize()
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for i in range(2) for a, b in zip(outs[i], want[i]))
    assert ql.lib().ql_gemm_status(None) == 0


def test_offsets_beyond_32_bits():
    """An H of more than 2^31 values: its last rows are what the same rows alone give."""
    M, I, K = 75000, 28672, 64
    if torch.cuda.mem_get_info()[0] < 12 << 30:
        pytest.skip("needs 12 GB")
    x = randn((M, K), torch.bfloat16, 8300)
    wg, wu = randn((I, K), torch.bfloat16, 8301, 0.125), randn((I, K), torch.bfloat16, 8302, 0.125)
    h = ql.gated_linear(x, wg, wu)
    tail = ql.gated_linear(x[-256:], wg, wu)
    assert torch.equal(h[-256:], tail)


def test_a_feed_forward_block_with_a_4_bit_down_projection():
    """The operators in a row, as a block uses them: the gated projection, its result quantized to MXFP4, the 4-bit down
    projection; and the fp8 block made of the same weights, which the 16-bit one is the yardstick of."""
    T, H, I = 48, 256, 512
    x = randn((T, H), torch.bfloat16, 8400)
    wg, wu, wd = randn((I, H), torch.bfloat16, 8401, H ** -0.5), randn((I, H), torch.bfloat16, 8402, H ** -0.5), randn((H, I), torch.bfloat16, 8403, I ** -0.5)
    h = ql.gated_linear(x, wg, wu)
    qd, sd = ql.quantize_mxfp4(wd)
    qh, sh = ql.quantize_mxfp4(h)
    y = ql.gemm_mxfp4(qh, sh, qd, sd)
    want = ql.dequantize_mxfp4(qh, sh).double() @ ql.dequantize_mxfp4(qd, sd).double().T
    assert torch.allclose(y.double(), want, rtol=2.0 ** -8, atol=1e-5)
    full = act_both(x.double() @ wg.double().T, "silu")[0] * (x.double() @ wu.double().T) @ wd.double().T
    rel = lambda a: float((a.double() - full).norm() / full.norm())
    # e2m1 keeps two significant bits: half a step is 1/8 to 1/4 of a value's binade, an rms of about a tenth for each operand
    assert rel(y) < 0.25
    # the 16-bit block's own error is its two roundings
    assert rel(h @ wd.t()) < 2.0 ** -7
    # fp8 weights and activations keep four: the block without its norm (x is put through one there), of unit rms rows
    xn = (x.double() / (x.double().pow(2).mean(dim=1, keepdim=True) + 1e-5).sqrt()).to(torch.bfloat16)
    hn = ql.gated_linear(xn, wg, wu)
    fp8 = ql.QuantizedMLP(wg, wu, wd)(x)
    ref = hn.double() @ wd.double().T
    assert float((fp8.double() - ref).norm() / ref.norm()) < 0.1


def test_refusals():
    x, w = torch.ones((4, 16), dtype=torch.bfloat16, device="cuda"), torch.ones((8, 16), dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ql.QlError, match="f16 or bf16"):
        ql.gated_linear(x.float(), w.float(), w.float())
    with pytest.raises(ql.QlError, match="of one type"):
        ql.gated_linear(x, w, w.half())
    with pytest.raises(ql.QlError, match="multiples of 8"):
        ql.gated_linear(x[:, :12], w[:, :12], w[:, :12])
    with pytest.raises(ql.QlError, match=r"must both be \[I,K\]"):
        ql.gated_linear(x, w, w[:4])
    with pytest.raises(ql.QuantizeError, match="out must have shape"):
        ql.gated_linear(x, w, w, out=torch.empty((4, 16), dtype=torch.bfloat16, device="cuda"))
    with pytest.raises(ql.QuantizeError, match="contiguous"):
        ql.gated_linear(x, w, w, out=torch.empty((8, 4), dtype=torch.bfloat16, device="cuda").t())
    with pytest.raises(ql.QlError, match="one device"):
        ql.gated_linear(x, w, w.cpu())
    with pytest.raises(ql.QuantizeError, match="leading dimensions"):
        ql.gated_linear_backward(torch.ones((5, 8), dtype=torch.bfloat16, device="cuda"), x, w, w)
    with pytest.raises(ql.QlError, match=r"grad must be \[M,I\]"):
        ql.gated_linear_backward(torch.ones((4, 16), dtype=torch.bfloat16, device="cuda"), x, w, w)
    with pytest.raises(ql.QlError, match="16-byte aligned"):
        ql.gated_linear(torch.ones(4 * 16 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(4, 16), w, w)


@pytest.mark.parametrize("M", [21, 300])
@pytest.mark.parametrize("activation", ["silu", "gelu", "gelu_tanh", "relu"])
def test_gates_of_every_size(activation, M):
    """One channel whose gate and up are values of x themselves, so that G and U are exact: gates from 2^-20 to 2^66, where a
    square is no f32 any more.  h is rounded once, dG and dU once and then again, unchanged, as the one term of dX's sum.  In
    f32 before that: a few ulp, of an exponential of up to 80 about 80 2^-23, far below the rounding's 2^-8; beyond 80 the true
    values are below 2^-110."""
    z = torch.tensor([s * v for v in (2.0 ** -20, 0.25, 1.0, 2.5, 6.0, 12.0, 40.0, 80.0, 2.0 ** 20, 2.0 ** 66) for s in (1, -1)] + [0.0])
    z = z.repeat(-(-M // len(z)))[:M].double()
    x, wg, wu = torch.zeros(M, 8, dtype=torch.bfloat16, device="cuda"), *torch.zeros(2, 8, 8, dtype=torch.bfloat16, device="cuda")
    x[:, 0], x[:, 1], wg[0, 0], wu[0, 1] = z.to(torch.bfloat16).cuda(), 1.5, 1.0, 1.0
    grad = torch.zeros(M, 8, dtype=torch.bfloat16, device="cuda")
    grad[:, 0] = 0.75
    z = x[:, 0].double().cpu()
    if activation == "silu":
        s = 1 / (1 + torch.exp(-z))
        a, d = z * s, s + z * s * (1 / (1 + torch.exp(z)))
    elif activation == "gelu":
        c = torch.special.erfc(-z / 2 ** 0.5) / 2
        a, d = z * c, c + z * torch.exp(-z * z / 2) / (2 * torch.pi) ** 0.5
    elif activation == "gelu_tanh":
        k = (2 / torch.pi) ** 0.5
        y = 2 * k * (z + 0.044715 * z ** 3)
        s = 1 / (1 + torch.exp(-y))
        a, d = z * s, s + torch.where(z.abs() < 1e3, z * s / (1 + torch.exp(y)) * 2 * k * (1 + 0.134145 * z * z), torch.zeros_like(z))
    else:
        a, d = z.clamp(min=0), (z > 0).double()
    h = ql.gated_linear(x, wg, wu, activation)[:, 0].double().cpu()
    dx = ql.gated_linear_backward(grad, x, wg, wu, activation, need_weight_grad=False)[0].double().cpu()
    close = lambda got, want: torch.allclose(got, want, rtol=2.0 ** -8 + 2.0 ** -12, atol=2.0 ** -108)
    assert close(h, 1.5 * a)
    assert close(dx[:, 0], 0.75 * 1.5 * d)
    assert close(dx[:, 1], 0.75 * a)


@pytest.mark.parametrize("M", [16, 300])
@pytest.mark.parametrize("activation", ["silu", "gelu", "gelu_tanh", "relu"])
def test_a_nan_weight_spoils_its_channel_only(activation, M):
    x, wg, wu = randn((M, 16), torch.float16, 8500), randn((24, 16), torch.float16, 8501, 0.25), randn((24, 16), torch.float16, 8502, 0.25)
    grad = randn((M, 24), torch.float16, 8503)
    wg[5, 3] = float("nan")
    h = ql.gated_linear(x, wg, wu, activation)
    _, dwg, dwu = ql.gated_linear_backward(grad, x, wg, wu, activation, need_input_grad=False)
    channel = torch.arange(24, device="cuda") == 5
    assert torch.equal(h.isnan(), channel.expand(M, 24))
    for g in (dwg, dwu):
        assert torch.equal(g.isnan(), channel[:, None].expand(24, 16))


# 33 to 128 tokens through more channels than one wave of 64 a CTA covers: below, at and above a token tile, channels with tails
@pytest.mark.parametrize("M,I,K", [(33, 9600, 136), (64, 11008, 520), (65, 10000, 72), (128, 18944, 264), (128, 12008, 1032), (100, 19000, 200)])
@pytest.mark.parametrize("dtype,act", [(torch.bfloat16, "silu"), (torch.float16, "gelu"), (torch.float16, "gelu_tanh"), (torch.bfloat16, "relu")])
def test_many_channels_of_few_tokens(M, I, K, dtype, act):
    test_forward(M, I, K, dtype, act)
    test_backward(M, I, K, dtype, act)


@pytest.mark.parametrize("M,I,K", [(1, 64, 64), (2, 264, 136), (16, 64, 128), (33, 64, 64), (40, 4104, 520), (100, 12000, 72), (128, 136, 1032)])
@pytest.mark.parametrize("dtype,act", [(torch.bfloat16, "silu"), (torch.float16, "gelu"), (torch.bfloat16, "relu")])
def test_few_tokens_gradients_are_rounded_once(M, I, K, dtype, act):
    """Up to 128 tokens the roundings of dG and dU are carried along: what is left is the last rounding, whose error is measured
    on the exact gradients.  Beside it stand the remainders' own roundings, 2^-8 of a rounding (f16: 2^-11, and for remainders
    below its normal range at most 2^-25 of absolute size against gradients of 0.01 and more), and f32 sums and functions, a
    few 2^-22: together below a twentieth of it."""
    c = [randn((M, K), dtype, 8600), randn((I, K), dtype, 8601, K ** -0.5), randn((I, K), dtype, 8602, K ** -0.5), randn((M, I), dtype, 8603)]
    x, wg, wu, d = [t.double() for t in c]
    g, u = x @ wg.T, x @ wu.T
    a, da = act_both(g, act)
    dg, du = d * u * da, d * a
    for got, want in zip(ql.gated_linear_backward(c[3], c[0], c[1], c[2], act), (dg @ wg + du @ wu, dg.T @ x, du.T @ x)):
        off, rounding = float((got.double() - want).norm()), float((want.to(dtype).double() - want).norm())
        assert off < 1.05 * rounding, f"{off / rounding:.3f} of one rounding"


def test_calls_from_several_threads_and_a_replayed_one():
    """Host threads on streams of their own, shapes of every kernel, while a captured backward pass is replayed beside them."""
    import threading
    shapes = [(1, 512, 264), (40, 9600, 136), (100, 264, 1032), (300, 1000, 328), (700, 2056, 264)]
    ops = [(randn((M, I), torch.bfloat16, 8700 + M), randn((M, K), torch.bfloat16, 8701 + M), randn((I, K), torch.bfloat16, 8702 + M, K ** -0.5),
            randn((I, K), torch.bfloat16, 8703 + M, K ** -0.5)) for M, I, K in shapes]
    want = [(ql.gated_linear(x, wg, wu), *ql.gated_linear_backward(d, x, wg, wu)) for d, x, wg, wu in ops]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        replayed = ql.gated_linear_backward(*ops[3])
    wrong = []

    def work(seed):
        with torch.cuda.stream(torch.cuda.Stream()):
            for k in range(10):
                i = (seed + k) % len(ops)
                d, x, wg, wu = ops[i]
                got = (ql.gated_linear(x, wg, wu), *ql.gated_linear_backward(d, x, wg, wu))
                torch.cuda.current_stream().synchronize()
                wrong.extend((i, j) for j, (a, b) in enumerate(zip(got, want[i])) if not torch.equal(a, b))
    threads = [threading.Thread(target=work, args=(s,)) for s in range(4)]
    for t in threads:
        t.start()
    for _ in range(20):
        graph.replay()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not wrong
    assert all(torch.equal(a, b) for a, b in zip(replayed, want[3][1:]))
    assert ql.lib().ql_gemm_status(None) == 0
