"""An activation's number beyond 32 bits is refused by the TVM-FFI entries, not cut down to one that exists."""
import os

import pytest
import torch

from conftest import ROOT

PLUGIN = os.path.join(ROOT, "tensorrt-incubator_b200", "lib", "libqlinear_b200_tvmffi.so")
tvm_ffi = pytest.importorskip("tvm_ffi")


@pytest.mark.gpu
@pytest.mark.parametrize("number", [1 << 32, (1 << 32) + 3, -(1 << 32), 4, -1])
def test_activation_beyond_32_bits(number):
    if not os.path.exists(PLUGIN):
        pytest.skip("plug-in not built")
    mod = tvm_ffi.load_module(PLUGIN)
    x, w, h = (torch.ones(s, dtype=torch.bfloat16, device="cuda") for s in ((4, 16), (8, 16), (4, 8)))
    with pytest.raises(Exception, match="unknown activation"):
        mod.ql_gated_linear(x, w, w, number, h)
    dx = torch.empty_like(x)
    scratch = torch.empty(mod.ql_gated_linear_backward_workspace(x, w, 1, 0), dtype=torch.uint8, device="cuda")
    with pytest.raises(Exception, match="unknown activation"):
        mod.ql_gated_linear_backward(h, x, w, w, number, dx, None, None, scratch)
