"""A process whose first call of an operator is a captured one: nothing the call sets up for itself (the device's status
word, kernel attributes, workspaces) may get in the way of the capture, and the replayed result is the eager call's."""
import os
import subprocess
import sys

import pytest

from conftest import ROOT

pytestmark = pytest.mark.gpu

PROGRAM = """
import sys
sys.path.insert(0, sys.argv[1])
import torch
import qlinear as ql
x = torch.randn(64, 544, device="cuda").bfloat16()
w = (torch.randn(256, 544, device="cuda") / 20).bfloat16()
grad = torch.randn(64, 256, device="cuda").bfloat16()
byte = lambda *shape, lo, hi: torch.randint(lo, hi, shape, device="cuda", dtype=torch.uint8)
f4 = lambda rows: (ql.Float4Tensor(byte(rows * 272, lo=0, hi=255), (rows, 544)), byte(rows, 17, lo=120, hi=130).view(torch.float8_e8m0fnu))
a, b = f4(64), f4(5000)
calls = {"quantize": lambda: ql.quantize_mxfp4(x)[1], "dequantize": lambda: ql.dequantize_mxfp4(*a), "product": lambda: ql.gemm_mxfp4(*a, *b),
         "gated": lambda: ql.gated_linear(x, w, w), "backward": lambda: ql.gated_linear_backward(grad, x, w, w)[1]}
call = calls[sys.argv[2]]
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    y = call()
g.replay()
torch.cuda.synchronize()
assert torch.equal(y.view(torch.uint8), call().view(torch.uint8))
assert ql.lib().ql_gemm_status(None) == 0
"""


@pytest.mark.parametrize("what", ["quantize", "dequantize", "product", "gated", "backward"])
def test_first_call_is_captured(what):
    r = subprocess.run([sys.executable, "-c", PROGRAM, os.path.join(ROOT, "tensorrt-incubator_b200"), what], capture_output=True, text=True, timeout=240)
    assert r.returncode == 0, r.stdout + r.stderr


@pytest.mark.parametrize("what", ["product", "gated"])
def test_first_call_is_captured_on_a_stream_that_synchronises_with_the_default_one(what):
    """Such a stream's capture ends where the process touches the default stream meanwhile."""
    program = PROGRAM.replace("g = torch.cuda.CUDAGraph()", """
import ctypes
rt, stream = ctypes.CDLL("libcudart.so.12"), ctypes.c_void_p()
assert rt.cudaStreamCreate(ctypes.byref(stream)) == 0
g = torch.cuda.CUDAGraph()""").replace("with torch.cuda.graph(g):", "with torch.cuda.graph(g, stream=torch.cuda.ExternalStream(stream.value)):")
    assert program.count("ExternalStream") == 1 and program.count("cudaStreamCreate") == 1
    r = subprocess.run([sys.executable, "-c", program, os.path.join(ROOT, "tensorrt-incubator_b200"), what], capture_output=True, text=True, timeout=240)
    assert r.returncode == 0, r.stdout + r.stderr
