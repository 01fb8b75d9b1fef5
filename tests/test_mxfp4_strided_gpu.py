"""Quantizing views that are not dense, and operands of the product cut out of larger ones."""
import pytest
import torch

import qlinear as ql
from helpers import randn
from test_mxfp4_gpu import check_quantized

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_views(dtype):
    base = randn((96, 512), dtype, 4100)
    turned = base.t()                                  # (512, 96), strides (1, 512)
    for view in (turned, turned[::3], base[:, 64:192], base[1::2, :32], base[:1].expand(5, 512), base.view(4, 24, 512).transpose(0, 1)):
        assert not view.is_contiguous()
        data, scales, _, _ = check_quantized(view)
        d2, s2 = ql.quantize_mxfp4(view.contiguous())
        assert torch.equal(data.packed, d2.packed) and torch.equal(scales.view(torch.uint8), s2.view(torch.uint8))
        back = ql.dequantize_mxfp4(data, scales, ql.float32)
        assert back.shape == view.shape
        # half a step of e2m1: at most 1 of a block's scale between 4 and 6, 2 beyond (saturation), of which m < 8 scales
        assert ((back - view.float()).abs() <= 2 * scales.float().repeat_interleave(32, dim=-1)).all()


def test_scales_cut_out_of_larger_ones():
    """Columns and rows of a larger matrix's scales: strided, and on odd addresses."""
    a, b = randn((40, 96), torch.bfloat16, 4110), randn((72, 96), torch.bfloat16, 4111)
    (qa, sa), (qb, sb) = ql.quantize_mxfp4(a), ql.quantize_mxfp4(b)
    want = ql.gemm_mxfp4(qa, sa, qb, sb, ql.float32)
    wide = torch.zeros((40, 7), dtype=torch.uint8, device="cuda")
    wide[:, 2:5] = sa.view(torch.uint8)
    whole = torch.zeros((1 + 72, 3), dtype=torch.uint8, device="cuda")
    whole[1:] = sb.view(torch.uint8)
    got = ql.gemm_mxfp4(qa, wide[:, 2:5].view(torch.float8_e8m0fnu), qb, whole[1:].view(torch.float8_e8m0fnu), ql.float32)
    assert torch.equal(got, want)
