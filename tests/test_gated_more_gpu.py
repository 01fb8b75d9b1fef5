"""The gated projection at an infinite gate, and gradients of 65 to 128 tokens where the roundings of dG and dU are not carried
along (more than 256 channels and columns)."""
import math

import pytest
import torch

import qlinear as ql
from helpers import randn
from test_gated_gpu import ACTS, Case, act_both, close

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("M", [4, 300])
def test_an_infinite_gate(act, M):
    """H is what the formula gives, NaN where an infinity meets a zero, and the other rows know nothing of it."""
    K = I = 64
    x = randn((M, K), torch.bfloat16, 8800)
    x[1] = 0
    x[1, 0] = float("inf")
    x[2] = 0
    x[2, 3] = -float("inf")
    eye = torch.eye(I, K, dtype=torch.bfloat16, device="cuda")
    want = act_both(x.double(), act)[0] * x.double()
    want[1, 1:] = want[2, :3] = want[2, 4:] = float("nan")   # infinity times the other weights' zeros
    h = ql.gated_linear(x, eye, eye, act)
    assert torch.equal(h.isnan(), want.isnan()) and float(h[1, 0]) == float("inf")
    rest = torch.arange(M, device="cuda") % M > 2
    assert torch.allclose(h[rest].double(), want[rest], rtol=2.0 ** -8 + 2.0 ** -12, atol=2.0 ** -100)


@pytest.mark.parametrize("M,I,K", [(65, 264, 264), (77, 1032, 520), (100, 1000, 520), (128, 512, 1032), (128, 4104, 264)])
@pytest.mark.parametrize("dtype,act", [(torch.bfloat16, "silu"), (torch.float16, "gelu"), (torch.bfloat16, "relu"), (torch.float16, "gelu_tanh")])
def test_gradients_of_65_to_128_tokens(M, I, K, dtype, act):
    """Each value within the worst case; all together within sqrt(2) of one rounding, measured on the exact gradients, with a
    quarter to spare."""
    c = Case(M, I, K, dtype, act, 8900 + M).exact()
    for got, (want, bound), name in zip(ql.gated_linear_backward(c.dh, c.x, c.wg, c.wu, act), (c.dx, c.dwg, c.dwu), ("dx", "dw_gate", "dw_up")):
        close(got, want, bound, f"{name} {M}x{I}x{K} {act}")
        off, one = float((got.double() - want).norm()), float((want.to(dtype).double() - want).norm())
        assert off < 1.25 * math.sqrt(2) * one, f"{name}: {off / one:.2f} roundings"
    assert ql.lib().ql_gemm_status(None) == 0
