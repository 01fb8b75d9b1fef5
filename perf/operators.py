"""Cases of the microscaled 4-bit operators and of the gated projection with its backward pass: what a pass computes, on
which sizes, and the plain form it is compared with.

    mx_round_trip   quantize_mxfp4 and dequantize_mxfp4: blocks of 32 along the last axis share a power of two
    mx_product      gemm_mxfp4: both operands in that form, one rounding of the f32 sums
    gated           gated_linear: act(x Wg^T) * (x Wu^T)
    gated_backward  gated_linear_backward: the gradients of x, Wg and Wu from the gradient of the result
"""
import math
import os
import sys

import torch

own = False

BLOCK = 32
_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
_LARGEST_PRODUCT = 8192 * 28672 * 8192
_LARGEST_GATED = 4096 * 28672 * 8192
_LARGEST_BACKWARD = 4096 * 11008 * 4096
_LARGEST_ROUND_TRIP = 8192 * 8192


def listed():
    return [
        # one token's hidden state, quantized before a 4-bit projection: all latency
        {"name": "round trip, one token", "op": "mx_round_trip", "rows": 1, "cols": 8192, "dtype": "bf16"},
        # f32 rows of an odd number, as exported weights come
        {"name": "round trip, odd f32 rows", "op": "mx_round_trip", "rows": 3063, "cols": 1184, "dtype": "f32"},
        # the activations of a long prompt
        {"name": "round trip, prompt", "op": "mx_round_trip", "rows": 8192, "cols": 8192, "dtype": "bf16"},
        # decoding one token through a wide projection: the weights are read once
        {"name": "product, one token", "op": "mx_product", "M": 1, "N": 28672, "K": 8192, "dtype": "bf16"},
        # a decoding batch
        {"name": "product, small batch", "op": "mx_product", "M": 24, "N": 4096, "K": 11008, "dtype": "f16"},
        # a ragged chunk of a prompt: no size is a multiple of a tile
        {"name": "product, ragged", "op": "mx_product", "M": 333, "N": 1001, "K": 2080, "dtype": "bf16"},
        # a long prompt through the widest projection
        {"name": "product, prompt", "op": "mx_product", "M": 8192, "N": 28672, "K": 8192, "dtype": "bf16"},
        # decoding one token
        {"name": "gated, one token", "op": "gated", "M": 1, "I": 11008, "K": 4096, "dtype": "bf16", "activation": "silu"},
        # a ragged batch through a small block
        {"name": "gated, ragged", "op": "gated", "M": 211, "I": 2744, "K": 1032, "dtype": "f16", "activation": "gelu"},
        # a long prompt through the widest block
        {"name": "gated, prompt", "op": "gated", "M": 4096, "I": 28672, "K": 8192, "dtype": "bf16", "activation": "silu"},
        # fine-tuning on a few short texts
        {"name": "backward, ragged", "op": "gated_backward", "M": 77, "I": 2744, "K": 1032, "dtype": "f16", "activation": "gelu_tanh"},
        # a training step's micro-batch
        {"name": "backward, training", "op": "gated_backward", "M": 4096, "I": 11008, "K": 4096, "dtype": "bf16", "activation": "silu"},
    ]


def _spread(rng, low, high, step=1):
    """A multiple of `step` in [low, high], spread over the logarithm."""
    v = math.exp(rng.uniform(math.log(low), math.log(high)))
    return min(high - high % step, max(step, low, int(round(v / step)) * step))


def draw(rng):
    op = rng.choice(["mx_round_trip", "mx_product", "gated", "gated_backward"])
    while True:
        if op == "mx_round_trip":
            case = {"op": op, "rows": _spread(rng, 1, 16384), "cols": _spread(rng, 32, 28672, 32), "dtype": rng.choice(["f32", "f16", "bf16"])}
            cost, most = case["rows"] * case["cols"], _LARGEST_ROUND_TRIP
        elif op == "mx_product":
            case = {"op": op, "M": _spread(rng, 1, 8192), "N": _spread(rng, 16, 28672), "K": _spread(rng, 32, 28672, 32), "dtype": rng.choice(["f32", "f16", "bf16"])}
            cost, most = case["M"] * case["N"] * case["K"], _LARGEST_PRODUCT
        else:
            case = {"op": op, "M": _spread(rng, 1, 8192), "I": _spread(rng, 64, 28672, 8), "K": _spread(rng, 64, 8192, 8), "dtype": rng.choice(["f16", "bf16"]),
                    "activation": rng.choice(["silu", "gelu", "gelu_tanh", "relu"])}
            cost, most = case["M"] * case["I"] * case["K"], _LARGEST_GATED if op == "gated" else _LARGEST_BACKWARD
        if cost <= most:
            return case


def _activations(shape, g):
    """Hidden states: normal, with channels that stand out."""
    channel = torch.exp(0.5 * torch.randn(shape[-1], generator=g, device="cuda"))
    return torch.randn(shape, generator=g, device="cuda") * channel


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dtype = _TYPES[case["dtype"]]
    state = {"case": case}
    if case["op"] == "mx_round_trip":
        state["x"] = _activations((case["rows"], case["cols"]), g).to(dtype)
        return state
    if case["op"] == "mx_product":
        a = _activations((case["M"], case["K"]), g)
        state["a"], state["a_scales"] = _pack(a)
        b = torch.randn((case["N"], case["K"]), generator=g, device="cuda") * case["K"] ** -0.5
        state["b"], state["b_scales"] = _pack(b)
        return state
    M, I, K = case["M"], case["I"], case["K"]
    state["x"] = torch.randn((M, K), generator=g, device="cuda").to(dtype)
    state["w_gate"] = (torch.randn((I, K), generator=g, device="cuda") * K ** -0.5).to(dtype)
    state["w_up"] = (torch.randn((I, K), generator=g, device="cuda") * K ** -0.5).to(dtype)
    if case["op"] == "gated_backward":
        state["grad"] = (torch.randn((M, I), generator=g, device="cuda") * 0.1).to(dtype)
    return state


# ---- the plain forms

def _block_scales(blocks):
    """2^(floor(log2 max|x|) - 2) of each block, 2^-127 at the least; NaN where the block holds an infinity or a NaN."""
    largest = blocks.abs().amax(dim=-1)
    exponent = torch.frexp(largest).exponent - 1          # largest = f * 2^e with 0.5 <= f < 1
    exponent = torch.where(largest > 0, exponent, torch.full_like(exponent, -200))
    scales = torch.ldexp(torch.ones_like(largest), (exponent - 2).clamp(min=-127))
    return torch.where(torch.isfinite(largest), scales, torch.full_like(scales, float("nan")))


def _codes(t):
    """The e2m1 code of |t|, nearest, ties to the even code, saturating."""
    t = t.abs()
    # between neighbours 0, .5, 1, 1.5, 2, 3, 4, 6 the border belongs to the even one of the two codes
    return ((t > 0.25).to(torch.uint8) + (t >= 0.75) + (t > 1.25) + (t >= 1.75) + (t > 2.5) + (t >= 3.5) + (t > 5.0)).to(torch.uint8)


def _quantized(x):
    """(values of e2m1 with their signs, scales) of f32 `x`."""
    blocks = x.reshape(x.shape[:-1] + (x.shape[-1] // BLOCK, BLOCK))
    scales = _block_scales(blocks)
    ratio = blocks / scales.unsqueeze(-1)
    codes = torch.where(torch.isnan(scales).unsqueeze(-1), torch.zeros_like(ratio, dtype=torch.uint8), _codes(ratio))
    return codes, torch.signbit(blocks), scales


def _pack(x):
    """What a 4-bit checkpoint holds: two codes a byte, the first in the low half, and the scales' exponents."""
    codes, negative, scales = _quantized(x)
    codes = (codes | (negative.to(torch.uint8) << 3)).reshape(-1, 2)
    return codes[:, 0] | (codes[:, 1] << 4), scales.to(torch.float8_e8m0fnu)


def _unpack(packed, shape):
    table = torch.tensor(_E2M1 + tuple(-v for v in _E2M1), dtype=torch.float32, device=packed.device)
    return table[torch.stack([packed & 15, packed >> 4], dim=-1).to(torch.int32)].reshape(shape)


def _activate(z, name):
    """(act(z), act'(z))"""
    if name == "silu":
        s = 1 / (1 + torch.exp(-z))
        return z * s, s * (1 + z * (1 - s))
    if name == "gelu":
        cdf = 0.5 * torch.erfc(-z * math.sqrt(0.5))
        return z * cdf, cdf + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    if name == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        t = torch.tanh(c * (z + 0.044715 * z * z * z))
        return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)
    return z.clamp(min=0), (z > 0).to(z.dtype)


def _plain(state):
    case = state["case"]
    dtype = _TYPES[case["dtype"]]
    if case["op"] == "mx_round_trip":
        codes, negative, scales = _quantized(state["x"].float())
        values = torch.tensor(_E2M1, dtype=torch.float32, device=codes.device)[codes.to(torch.int32)]
        values = torch.where(negative, -values, values) * scales.unsqueeze(-1)
        return {"values": values.reshape(state["x"].shape).to(dtype), "scales": scales.to(torch.float8_e8m0fnu)}
    if case["op"] == "mx_product":
        a = _unpack(state["a"], state["a_scales"].shape + (BLOCK,)) * state["a_scales"].float().unsqueeze(-1)
        b = _unpack(state["b"], state["b_scales"].shape + (BLOCK,)) * state["b_scales"].float().unsqueeze(-1)
        return torch.matmul(a.reshape(case["M"], case["K"]), b.reshape(case["N"], case["K"]).t()).to(dtype)
    x, w_gate, w_up = state["x"].float(), state["w_gate"].float(), state["w_up"].float()
    gate, up = torch.matmul(x, w_gate.t()), torch.matmul(x, w_up.t())
    act, slope = _activate(gate, case["activation"])
    if case["op"] == "gated":
        return (act * up).to(dtype)
    grad = state["grad"].float()
    d_gate, d_up = grad * up * slope, grad * act
    return {"x": (torch.matmul(d_gate, w_gate) + torch.matmul(d_up, w_up)).to(dtype),
            "w_gate": torch.matmul(d_gate.t(), x).to(dtype), "w_up": torch.matmul(d_up.t(), x).to(dtype)}


# ---- the framework's operators

def _own(state):
    package = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tensorrt-incubator_b200")
    if package not in sys.path:
        sys.path.insert(0, package)
    import qlinear as ql

    case = state["case"]
    out = {"f32": ql.float32, "f16": ql.float16, "bf16": ql.bfloat16}[case["dtype"]]
    if case["op"] == "mx_round_trip":
        data, scales = ql.quantize_mxfp4(state["x"])
        return {"values": ql.dequantize_mxfp4(data, scales, out), "scales": scales}
    if case["op"] == "mx_product":
        a = ql.Float4Tensor(state["a"], (case["M"], case["K"]))
        b = ql.Float4Tensor(state["b"], (case["N"], case["K"]))
        return ql.gemm_mxfp4(a, state["a_scales"], b, state["b_scales"], out_dtype=out)
    if case["op"] == "gated":
        return ql.gated_linear(state["x"], state["w_gate"], state["w_up"], case["activation"])
    x, w_gate, w_up = ql.gated_linear_backward(state["grad"], state["x"], state["w_gate"], state["w_up"], case["activation"])
    return {"x": x, "w_gate": w_gate, "w_up": w_up}


def run(state):
    return _own(state) if own else _plain(state)


def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "mx_round_trip":
        n = case["rows"] * case["cols"]
        # x in, data and scales out; data and scales in, values out
        return {"bytes": 2 * (n * size + n / 2 + n / 32), "flops": 4 * n}
    if case["op"] == "mx_product":
        M, N, K = case["M"], case["N"], case["K"]
        return {"bytes": (M + N) * K * (1 / 2 + 1 / 32) + M * N * size, "flops": 2 * M * N * K}
    M, I, K = case["M"], case["I"], case["K"]
    if case["op"] == "gated":
        return {"bytes": size * (M * K + 2 * I * K + M * I), "flops": 4 * M * I * K}
    return {"bytes": size * (2 * M * K + 4 * I * K + M * I), "flops": 12 * M * I * K}


# ---- the definitions in 64 bits

def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "mx_round_trip":
        x = state["x"].double()
        lead = x.shape[:-1]
        x = x.reshape(*lead, -1, BLOCK)
        top = x.abs().max(dim=-1, keepdim=True).values
        # the largest power of two that is no larger than the largest value, a quarter of it: found by comparison, not by logarithms
        powers = torch.pow(torch.tensor(2.0, dtype=torch.float64, device=x.device), torch.arange(-149, 128, dtype=torch.float64, device=x.device))
        at = torch.searchsorted(powers, top.reshape(-1), right=True).reshape(top.shape) - 1
        scale = torch.where(top > 0, powers[at.clamp(min=0)] / 4, torch.zeros_like(top)).clamp(min=2.0 ** -127)
        bad = ~torch.isfinite(top)
        # the grid of e2m1: steps of 1/2 below 2, of 1 below 4, of 2 above; torch.round goes to the even multiple
        t = (x / scale).abs()
        step = torch.where(t < 2, 0.5, torch.where(t < 4, 1.0, 2.0)).double()
        value = (torch.round(t / step) * step).clamp(max=6.0) * torch.sign(x) * scale
        nan = torch.full_like(value, float("nan"))
        return {"values": torch.where(bad, nan, value).reshape(*lead, -1), "scales": torch.where(bad, torch.full_like(scale, float("nan")), scale).squeeze(-1)}
    if case["op"] == "mx_product":
        def wide(packed, scales):
            code = torch.stack([packed.bitwise_and(15), packed.bitwise_right_shift(4)], dim=1).reshape(scales.shape[0], -1).short()
            e, m = (code >> 1) & 3, (code & 1).double()
            size = torch.where(e == 0, m / 2, torch.pow(2.0, (e - 1).double()) * (1 + m / 2))
            size = torch.where(code >= 8, -size, size)
            size *= torch.pow(2.0, scales.view(torch.uint8).double() - 127).repeat_interleave(BLOCK, dim=1)
            return size
        return wide(state["a"], state["a_scales"]) @ wide(state["b"], state["b_scales"]).T
    x, wg, wu = (state[k].double() for k in ("x", "w_gate", "w_up"))
    g, u = x @ wg.T, x @ wu.T
    kind = case["activation"]
    if kind == "silu":
        sg = torch.sigmoid(g)
        f, df = g * sg, sg + g * sg * (1 - sg)
    elif kind == "gelu":
        phi = (1 + torch.erf(g / 2 ** 0.5)) / 2
        f, df = g * phi, phi + g * torch.exp(-g ** 2 / 2) / (2 * math.pi) ** 0.5
    elif kind == "gelu_tanh":
        inner = (2 / math.pi) ** 0.5 * (g + 0.044715 * g ** 3)
        d_inner = (2 / math.pi) ** 0.5 * (1 + 0.134145 * g ** 2)
        f, df = g * (1 + inner.tanh()) / 2, (1 + inner.tanh()) / 2 + g / 2 * d_inner / inner.cosh() ** 2
    else:
        f, df = torch.relu(g), (g > 0).double()
    if case["op"] == "gated":
        return f * u
    dh = state["grad"].double()
    dg, du = dh * u * df, dh * f
    return {"x": dg @ wg + du @ wu, "w_gate": dg.T @ x, "w_up": du.T @ x}
