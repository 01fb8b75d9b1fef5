"""Gradients of every size through the 16-bit backward pass.  dG and dU stand in float16 between its kernels, whose range ends
at 65504 and whose digits fade below 2^-14; the gradients of x and the weights must not suffer from that.

Bounds, as in the other tests of the gated projection: up to 64 tokens the last rounding alone is left, with a twentieth for f32
sums and functions and for remainders of remainders; of more tokens the roundings of dG and dU come on top, averaged over many
values: sqrt(2) of one rounding, with a quarter to spare.  One rounding is measured on the exact gradients, so that results
below float16's normal range count with the rounding they have there."""
import math

import pytest
import torch

import qlinear as ql
from helpers import randn
from test_gated_gpu import act_both

pytestmark = pytest.mark.gpu


def exact(dh, x, wg, wu, act):
    dh, x, wg, wu = (t.double() for t in (dh, x, wg, wu))
    g, u = x @ wg.T, x @ wu.T
    a, d = act_both(g, act)
    dg, du = dh * u * d, dh * a
    return (dg @ wg + du @ wu, dg.T @ x, du.T @ x), max(float(dg.abs().max()), float(du.abs().max()))


def operands(M, I, K, seed, dh=1.0, x=1.0, wg=1.0, wu=1.0):
    f = torch.float16
    return (randn((M, I), f, seed, dh), randn((M, K), f, seed + 1, x), randn((I, K), f, seed + 2, wg * K ** -0.5), randn((I, K), f, seed + 3, wu * K ** -0.5))


def roundings(got, want):
    off, one = float((got.double() - want).norm()), float((want.to(got.dtype).double() - want).norm())
    return off / one


def check(tensors, act, want, M, **need):
    got = ql.gated_linear_backward(*tensors, act, **need)
    assert ql.lib().ql_gemm_status(None) == 0
    limit = 1.05 if M <= 64 else 1.25 * math.sqrt(2)
    for g, w, name in zip(got, want, ("dx", "dw_gate", "dw_up")):
        if g is not None:
            assert torch.isfinite(g).all(), name
            assert roundings(g, w) < limit, f"{name}: {roundings(g, w):.2f} roundings"
    return got


# each form of the first stage: cluster split, wide split, pairs of 64 and of 128 channels
SHAPES = [(1, 2744, 1032), (16, 2744, 1032), (64, 11008, 520), (77, 2744, 1032), (512, 1000, 328), (700, 2056, 1544)]


@pytest.mark.parametrize("M,I,K", SHAPES)
@pytest.mark.parametrize("std", [1e-4, 2.0 ** -16, 2e-6])
@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_small_gradients(M, I, K, std, act):
    t = operands(M, I, K, 9000 + M, dh=std)
    want, _ = exact(*t, act)
    got = check(t, act, want, M)
    assert all(torch.equal(a, b) for a, b in zip(got, ql.gated_linear_backward(*t, act)))
    check(t, act, want, M, need_weight_grad=False)
    check(t, act, want, M, need_input_grad=False)


@pytest.mark.parametrize("M,I,K", SHAPES)
def test_large_gradients_with_sums_in_range(M, I, K):
    """dG beyond 65504 throughout, the gradients of x and the weights well below it."""
    t = operands(M, I, K, 9100 + M, dh=4000.0, x=2.0 ** -10, wg=0.02, wu=30000.0)
    want, largest = exact(*t, "silu")
    assert largest > 4 * 65504 and all(torch.isfinite(w.half()).all() for w in want)
    check(t, "silu", want, M)


@pytest.mark.parametrize("M", [40, 300])
def test_tokens_of_unlike_gradients(M):
    """Every second token's gradient 2^-9 of the others': its row of dX has its own bound."""
    t = operands(M, 1000, 520, 9200 + M)
    t[0][1::2] *= 2.0 ** -9
    want, _ = exact(*t, "silu")
    dx, dwg, dwu = check(t, "silu", want, M)
    assert roundings(dx[1::2], want[0][1::2]) < (1.05 if M <= 64 else 1.25 * math.sqrt(2))


@pytest.mark.parametrize("M", [12, 40, 100, 300])
def test_infinities_and_zeros(M):
    """A gradient that is no number spoils its token's dX and its channel's weight gradients, and decides nothing for the others."""
    I, K = 264, 136
    t = operands(M, I, K, 9300 + M, dh=1e-5)
    t[0][5, 7], t[0][6, 9] = float("nan"), float("inf")
    got = ql.gated_linear_backward(*t, "silu")
    clean = t[0].clone()
    clean[5, 7] = clean[6, 9] = 0
    want, _ = exact(clean, *t[1:], "silu")
    limit = 1.05 if M <= 64 else 1.25 * math.sqrt(2)
    rows, channels = torch.ones(M, dtype=torch.bool, device="cuda"), torch.ones(I, dtype=torch.bool, device="cuda")
    rows[5] = rows[6] = channels[7] = channels[9] = False
    for g, w, keep in zip(got, want, (rows, channels, channels)):
        assert not torch.isfinite(g[~keep]).any() and torch.isfinite(g[keep]).all()
        assert roundings(g[keep], w[keep]) < limit
    for g in ql.gated_linear_backward(torch.zeros_like(clean), *t[1:], "silu"):
        assert not g.any()


@pytest.mark.parametrize("M", [8, 90, 400])
def test_replayed_with_gradients_of_other_sizes(M):
    """The choice is made on the device, on every replay."""
    t = operands(M, 520, 264, 9400 + M)
    dh = t[0].clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = ql.gated_linear_backward(*t, "silu")
    for std in (1.0, 1e-5, 300.0, 2e-6, 1.0):
        t[0].copy_((dh.double() * std).half())
        g.replay()
        torch.cuda.synchronize()
        want, _ = exact(*t, "silu")
        assert all(torch.equal(a, b) for a, b in zip(out, ql.gated_linear_backward(*t, "silu")))
        for got, w in zip(out, want):
            assert roundings(got, w) < (1.05 if M <= 64 else 1.25 * math.sqrt(2))
