"""The microscaled 4-bit layer, its input's gradient, and the root-mean-square norm with the residual's addition, as
measured cases.

One case is one pass of a program that serves a block in 4 bits, or trains what lies around its frozen 4-bit weights:

* ``linear``      ``mxfp4_linear``: activations quantized by 1 x 32 blocks, a weight held the same way, one float32 sum
                  per output, the bias added and the result rounded once;
* ``backward``    ``mxfp4_linear_backward``: the input's gradient through the frozen weight and the bias's, from the
                  output's gradient as it is;
* ``checkpoint``  ``quantize_mxfp4`` and ``dequantize_mxfp4``: an activation put away in 4 bits and taken out again;
* ``norm``        ``rms_norm`` with the residual added first, its output in the input's type, or quantized for the 8-bit
                  or the 4-bit layer (``rms_norm_quantize_fp8``, ``rms_norm_quantize_mxfp4``), restored here to the
                  values that it stands for;
* ``norm_grad``   ``rms_norm_backward``: the gradients of input and weight, from the normed input itself or as it was kept
                  in 8 bits, with the gradient that reaches the residual stream beside the norm.

Layer sizes are those of ``bench.py``'s workloads (hidden 5120 with a 20480 FFN, hidden 5376 with QKV 21504 and a
14336 SwiGLU) and generic odd ones; token counts run from one to the 75600 of 720p x 5 s.
"""

from __future__ import annotations

import math
import os
import sys

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_BYTES = {"bf16": 2, "f16": 2, "f32": 4}
_EPS = 1e-6

_LAYERS = ((5120, 5120), (5120, 20480), (20480, 5120), (5376, 21504), (14336, 5376))


def _mx():
    path = os.path.join(os.getcwd(), "x-minimaxh3_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import mx_qlinear

    return mx_qlinear


# ---------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------

def listed():
    return [
        # one token through the FFN's up projection: the smallest product, a stream of the weight
        {"name": "linear_one_token", "kind": "linear", "m": 1, "k": 5120, "n": 20480, "dtype": "bf16", "bias": True},
        # a 333-token prompt through a layer of odd sizes, float16
        {"name": "linear_ragged", "kind": "linear", "m": 333, "k": 5000, "n": 2049, "dtype": "f16", "bias": True},
        # a slab of 8192 tokens through the QKV projection
        {"name": "linear_slab", "kind": "linear", "m": 8192, "k": 5376, "n": 21504, "dtype": "bf16", "bias": False},
        # a square layer over a whole 720p clip
        {"name": "linear_720p", "kind": "linear", "m": 75600, "k": 5120, "n": 5120, "dtype": "bf16", "bias": True},
        # one step's input gradient through a layer of odd sizes, float16
        {"name": "backward_ragged", "kind": "backward", "m": 1501, "k": 1000, "n": 3001, "dtype": "f16"},
        # one step's input gradient through the SwiGLU's down projection over a slab of 8192 tokens
        {"name": "backward_slab", "kind": "backward", "m": 8192, "k": 14336, "n": 5376, "dtype": "bf16"},
        # float32 activations of an odd width put away and taken out
        {"name": "checkpoint_ragged", "kind": "checkpoint", "m": 1003, "k": 4999, "dtype": "f32"},
        # the FFN's hidden activations of a slab put away and taken out
        {"name": "checkpoint_slab", "kind": "checkpoint", "m": 8192, "k": 20480, "dtype": "bf16"},
        # one token's norm behind a residual addition: latency
        {"name": "norm_one_token", "kind": "norm", "m": 1, "d": 5120, "dtype": "bf16", "out": "same", "residual": True},
        # the norm of a whole 720p clip behind a residual addition, quantized for the 4-bit layer
        {"name": "norm_720p", "kind": "norm", "m": 75600, "d": 5376, "dtype": "bf16", "out": "mxfp4", "residual": True},
        # gradients at odd sizes in float32
        {"name": "norm_grad_ragged", "kind": "norm_grad", "m": 777, "d": 1003, "dtype": "f32", "kept": False, "residual": False},
        # gradients of a whole 720p clip, the input kept in 8 bits, the residual stream's gradient added
        {"name": "norm_grad_720p", "kind": "norm_grad", "m": 75600, "d": 5120, "dtype": "bf16", "kept": True, "residual": True},
    ]


def _spread(rng, lo, hi):
    """A whole number spread evenly over the logarithm of [lo, hi]."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("linear", "linear", "linear", "backward", "backward", "checkpoint", "norm", "norm", "norm_grad"))
    dtype = rng.choice(("bf16", "bf16", "f16", "f32"))
    if kind in ("linear", "backward"):
        if rng.random() < 0.5:
            k, n = rng.choice(_LAYERS)
        else:
            k, n = _spread(rng, 64, 8192), _spread(rng, 64, 8192)
        # no more work than the largest listed case of the kind
        top = 75600 * 5120 * 5120 if kind == "linear" else 8192 * 14336 * 5376 // 3
        m = _spread(rng, 1, max(1, min(75600, top // (k * n))))
        case = {"kind": kind, "m": m, "k": k, "n": n, "dtype": dtype}
        if kind == "linear":
            case["bias"] = rng.random() < 0.6
        return case
    d = _spread(rng, 8, 20480)
    m = _spread(rng, 1, min(75600, 75600 * 5120 // (2 * d)))
    if kind == "checkpoint":
        return {"kind": kind, "m": min(m, max(1, 8192 * 20480 // (2 * d))), "k": d, "dtype": dtype}
    case = {"kind": kind, "m": m, "d": d, "dtype": dtype}
    if kind == "norm":
        case["out"] = rng.choice(("same", "fp8", "mxfp4"))
    else:
        case["kept"] = rng.random() < 0.5
    case["residual"] = rng.random() < 0.5
    return case


# ---------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _activations(g, m, k, dtype):
    """Transformer activations: unit normal, 0.5 % of the channels 20 times larger."""
    x = torch.randn(m, k, generator=g, device="cuda")
    idx = torch.randperm(k, generator=g, device="cuda")[: -(-k * 5 // 1000)]
    x[:, idx] *= 20.0
    return x.to(dtype)


def _gradient(g, m, n, dtype):
    """An output's gradient: normal, small, tokens of different magnitude."""
    size = torch.exp(torch.randn(m, 1, generator=g, device="cuda"))
    return (torch.randn(m, n, generator=g, device="cuda") * size * 1e-2).to(dtype)


def _vec(g, n, mean, std, dtype):
    return (mean + torch.randn(n, generator=g, device="cuda") * std).to(dtype)


def prepare(case, seed):
    g = _gen(seed)
    kind, dtype = case["kind"], _DTYPES[case["dtype"]]
    state = {"case": case}
    if kind in ("linear", "backward"):
        m, k, n = case["m"], case["k"], case["n"]
        state["wq"], state["ws"] = _codes4(torch.randn(n, k, generator=g, device="cuda") * 0.02)
        if kind == "linear":
            state["x"] = _activations(g, m, k, dtype)
            state["bias"] = _vec(g, n, 0.0, 0.1, dtype) if case["bias"] else None
        else:
            state["dy"] = _gradient(g, m, n, dtype)
        if own:  # the layer's weight as a program keeps it
            state["weight"] = _mx().prepare_mxfp4_weight(state["wq"].view(torch.float4_e2m1fn_x2), state["ws"], in_features=k)
    elif kind == "checkpoint":
        state["x"] = _activations(g, case["m"], case["k"], dtype)
    else:
        m, d = case["m"], case["d"]
        x = _activations(g, m, d, dtype)
        state["weight"] = _vec(g, d, 1.0, 0.2, dtype)
        if kind == "norm":
            state["x"] = x
            state["residual"] = _activations(g, m, d, dtype) if case["residual"] else None
        else:
            state["rstd"] = (x.double().square().mean(1) + _EPS).rsqrt().float()
            state["dy"] = _gradient(g, m, d, dtype)
            state["dsum"] = _gradient(g, m, d, dtype) if case["residual"] else None
            if case["kept"]:
                state["xq"], state["xs"] = _codes8(x)
            else:
                state["x"] = x
    return state


# ---------------------------------------------------------------------------------------
# plain form
# ---------------------------------------------------------------------------------------

def _blocks(x, width):
    """x [M, K] in float32, zero-padded, as [M, blocks, width]."""
    m, k = x.shape
    x = x.float()
    if k % width:
        x = torch.nn.functional.pad(x, (0, -k % width))
    return x.view(m, -1, width)


def _pow2(e):
    return torch.ldexp(torch.ones_like(e, dtype=torch.float32), e)


def _exponents(absmax, top, least):
    """The smallest e >= least with absmax <= top * 2^e, 0 for a block of zeros."""
    mant, e = torch.frexp(absmax)
    top_mant, top_e = math.frexp(top)
    e = torch.where(mant > top_mant, e + 1, e) - top_e
    return torch.where(absmax == 0, torch.zeros_like(e), e.clamp(least, 127))


def _magnitude_codes(v):
    """Magnitudes up to 6 to the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 by number, ties to the even one."""
    return ((v > 0.25).to(torch.uint8) + (v >= 0.75).to(torch.uint8) + (v > 1.25).to(torch.uint8) + (v >= 1.75).to(torch.uint8)
            + (v > 2.5).to(torch.uint8) + (v >= 3.5).to(torch.uint8) + (v > 5.0).to(torch.uint8))


def _codes4(x):
    """x [M, K] -> (two e2m1 codes per byte uint8 [M, ceil(K / 2)], the even column's in the low four bits; scale e8m0
    [M, ceil(K / 32)])."""
    m, k = x.shape
    b = _blocks(x, 32)
    e = _exponents(b.abs().amax(-1), 6.0, -125)
    b = b * _pow2(-e)[..., None]
    c = (_magnitude_codes(b.abs()) + (b < 0).to(torch.uint8) * 8).view(m, -1, 2)
    q = (c[..., 0] + c[..., 1] * 16)[:, : -(-k // 2)].contiguous()
    return q, (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def _values4(q, s, k):
    """The float32 values of two codes per byte."""
    m = q.shape[0]
    c = torch.stack((q & 15, q >> 4), -1).view(m, -1)[:, :k]
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=q.device)
    v = table[(c & 7).long()] * torch.where(c > 7, -1.0, 1.0)
    return v * _pow2(s.view(torch.uint8).int() - 127).repeat_interleave(32, 1)[:, :k]


def _held4(x):
    """The float32 values that x stands for in 4 bits."""
    m, k = x.shape
    b = _blocks(x, 32)
    e = _exponents(b.abs().amax(-1), 6.0, -125)
    b = b * _pow2(-e)[..., None]
    c = _magnitude_codes(b.abs()).float()
    v = torch.where(c <= 4, c * 0.5, torch.where(c == 7, 6.0, c - 2.0))
    return (torch.copysign(v, b) * _pow2(e)[..., None]).view(m, -1)[:, :k]


def _codes8(x):
    """x [M, K] -> (q e4m3 [M, K], scale e8m0 [M, ceil(K / 128)]), one scale per row and 128 columns."""
    m, k = x.shape
    b = _blocks(x, 128)
    e = _exponents(b.abs().amax(-1), 448.0, -117)
    q = (b * _pow2(-e)[..., None]).to(torch.float8_e4m3fn)
    return q.view(m, -1)[:, :k].contiguous(), (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def _values8(q, s):
    return q.float() * _pow2(s.view(torch.uint8).int() - 127).repeat_interleave(128, 1)[:, : q.shape[1]]


def _plain(state):
    case = state["case"]
    kind, dtype = case["kind"], _DTYPES[case["dtype"]]
    if kind == "linear":
        y = _held4(state["x"]) @ _values4(state["wq"], state["ws"], case["k"]).t()
        if state["bias"] is not None:
            y = y + state["bias"].float()
        return y.to(dtype)
    if kind == "backward":
        dy = state["dy"]
        dx = dy.float() @ _values4(state["wq"], state["ws"], case["k"])
        return {"dx": dx.to(dtype), "dbias": dy.sum(0, dtype=torch.float64).float()}
    if kind == "checkpoint":
        return _held4(state["x"]).to(dtype)
    if kind == "norm":
        s = state["x"] if state["residual"] is None else (state["x"].float() + state["residual"].float()).to(dtype)
        # (in 64 bits: codes of 4 and 8 bits are values next to a border)
        rstd = (s.double().square().mean(1) + _EPS).rsqrt().float()
        y = s.float() * rstd[:, None] * state["weight"].float()
        y = y.to(dtype) if case["out"] == "same" else (_held4(y) if case["out"] == "mxfp4" else _values8(*_codes8(y))).to(torch.bfloat16)
        return {"y": y, "rstd": rstd} if state["residual"] is None else {"y": y, "sum": s, "rstd": rstd}
    x = _values8(state["xq"], state["xs"]) if case["kept"] else state["x"].float()
    xh = x * state["rstd"][:, None]
    dy = state["dy"].float()
    g = dy * state["weight"].float()
    dx = (g - xh * (g * xh).mean(1, keepdim=True)) * state["rstd"][:, None]
    if state["dsum"] is not None:
        dx = dx + state["dsum"].float()
    return {"dx": dx.to(dtype), "dweight": (dy * xh).sum(0, dtype=torch.float64).float()}


def run(state):
    if not own:
        return _plain(state)
    mx, case = _mx(), state["case"]
    kind = case["kind"]
    if kind == "linear":
        return mx.mxfp4_linear(state["x"], state["weight"], state["bias"])
    if kind == "backward":
        dx, db = mx.mxfp4_linear_backward(state["dy"], state["weight"])
        return {"dx": dx, "dbias": db}
    if kind == "checkpoint":
        q, s = mx.quantize_mxfp4(state["x"])
        return mx.dequantize_mxfp4(q, s, state["x"].dtype, width=case["k"])
    if kind == "norm":
        x, w, r = state["x"], state["weight"], state["residual"]
        if case["out"] == "same":
            y, *rest = mx.rms_norm(x, w, _EPS, residual=r, return_rstd=True)
        elif case["out"] == "fp8":
            q, s, *rest = mx.rms_norm_quantize_fp8(x, w, _EPS, residual=r, return_rstd=True)
            y = mx.dequantize_fp8_block128(q, s)
        else:
            q, s, *rest = mx.rms_norm_quantize_mxfp4(x, w, _EPS, residual=r, return_rstd=True)
            y = mx.dequantize_mxfp4(q, s, width=case["d"])
        return {"y": y, "rstd": rest[0]} if r is None else {"y": y, "sum": rest[0], "rstd": rest[1]}
    x = (state["xq"], state["xs"]) if case["kept"] else state["x"]
    dx, dw = mx.rms_norm_backward(state["dy"], x, state["rstd"], state["weight"], dsum=state["dsum"])
    return {"dx": dx, "dweight": dw}


# ---------------------------------------------------------------------------------------
# work and 64-bit values
# ---------------------------------------------------------------------------------------

def _held_bytes(m, k, out):
    """Bytes of a quantized [m, k]."""
    return m * (-(-k // 2) + -(-k // 32)) if out == "mxfp4" else m * (k + -(-k // 128))


def work(case):
    kind, e, m = case["kind"], _BYTES[case["dtype"]], case["m"]
    if kind in ("linear", "backward"):
        k, n = case["k"], case["n"]
        weight = _held_bytes(n, k, "mxfp4")
        if kind == "linear":
            bias = n * e if case["bias"] else 0
            return {"bytes": m * k * e + weight + bias + m * n * e, "flops": 2 * m * n * k}
        return {"bytes": m * n * e + weight + m * k * e + n * 4, "flops": 2 * m * n * k + m * n}
    if kind == "checkpoint":
        k = case["k"]
        return {"bytes": 2 * m * k * e + _held_bytes(m, k, "mxfp4"), "flops": 3 * m * k}
    d = case["d"]
    if kind == "norm":
        streams = 3 if case["residual"] else 1  # x, and with a residual that and the sum
        y = m * d * e if case["out"] == "same" else _held_bytes(m, d, case["out"]) + m * d * 2
        return {"bytes": streams * m * d * e + y + d * e + 4 * m, "flops": 5 * m * d}
    x = _held_bytes(m, d, "fp8") if case["kept"] else m * d * e
    streams = 3 if case["residual"] else 2  # dy, dx, and with a residual the stream's gradient
    return {"bytes": x + streams * m * d * e + 4 * m + d * e + 4 * d, "flops": 9 * m * d}


def _settled(top, most, least):
    """The smallest 2^e (e >= least) with top <= most * 2^e, found by log2 and settled by comparison."""
    scale = torch.exp2(torch.ceil(torch.log2(top / most)).clamp(least, 127))
    scale = torch.where(top == 0, torch.ones_like(scale), scale)
    scale = torch.where(top > most * scale, scale * 2, scale)
    return torch.where((top != 0) & (top <= most * scale / 2) & (scale > 2.0**least), scale / 2, scale)


def _round_e2m1(v):
    """float64 of magnitude up to 6 to the nearest e2m1 value, ties to even."""
    a = v.abs()
    step = torch.where(a < 2.0, 0.5, torch.where(a < 4.0, 1.0, 2.0))
    return torch.round(v / step) * step


def _round_e4m3(v):
    """float64 of magnitude up to 448 to the nearest e4m3 value, ties to even."""
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0**-6))) - 3)
    return torch.round(v / step) * step


def _held64(x, out):
    """The float64 values that x stands for, in slices of columns."""
    width, most, least, to = (32, 6.0, -125, _round_e2m1) if out == "mxfp4" else (128, 448.0, -117, _round_e4m3)
    m, k = x.shape
    y = torch.empty((m, k), dtype=torch.float64, device=x.device)
    for a in range(0, k, 1024):
        part = x[:, a : a + 1024].double()
        n = part.shape[1]
        part = torch.nn.functional.pad(part, (0, -n % width)).view(m, -1, width)
        scale = _settled(part.abs().amax(-1), most, least)[..., None]
        y[:, a : a + n] = (to(part / scale) * scale).view(m, -1)[:, :n]
    return y


def _stored64(q, s, k):
    """The float64 values of a stored weight."""
    low, high = (q % 16).long(), (q // 16).long()
    table = torch.tensor([0, 1, 2, 3, 4, 6, 8, 12, 0, -1, -2, -3, -4, -6, -8, -12], dtype=torch.float64, device=q.device) / 2
    v = torch.empty((q.shape[0], 2 * q.shape[1]), dtype=torch.float64, device=q.device)
    v[:, 0::2], v[:, 1::2] = table[low], table[high]
    f = torch.exp2(s.view(torch.uint8).double() - 127)
    v = v[:, :k]
    for b in range(f.shape[1]):
        v[:, b * 32 : (b + 1) * 32] *= f[:, b : b + 1]
    return v


def exact(case, seed):
    global own
    kind, dtype = case["kind"], _DTYPES[case["dtype"]]
    was, own = own, False
    try:
        state = prepare(case, seed)
    finally:
        own = was
    if kind == "linear":
        y = _held64(state["x"], "mxfp4") @ _stored64(state["wq"], state["ws"], case["k"]).t()
        return y if state["bias"] is None else y.add_(state["bias"].double())
    if kind == "backward":
        dy = state["dy"].double()
        return {"dx": dy @ _stored64(state["wq"], state["ws"], case["k"]), "dbias": dy.sum(0)}
    if kind == "checkpoint":
        return _held64(state["x"], "mxfp4")
    if kind == "norm":
        # (the sum is held in the input's type: what is normed is the rounded one)
        s = state["x"] if state["residual"] is None else (state["x"].double() + state["residual"].double()).to(dtype)
        s = s.double()
        rstd = 1.0 / (s.square().mean(1) + _EPS).sqrt()
        y = s * rstd[:, None] * state["weight"].double()
        if case["out"] != "same":
            y = _held64(y, case["out"])
        return {"y": y, "rstd": rstd} if state["residual"] is None else {"y": y, "sum": s, "rstd": rstd}
    if case["kept"]:
        x = state["xq"].to(torch.float32).double()
        f = torch.exp2(state["xs"].view(torch.uint8).double() - 127)
        for b in range(f.shape[1]):
            x[:, b * 128 : (b + 1) * 128] *= f[:, b : b + 1]
    else:
        x = state["x"].double()
    r = state["rstd"].double()[:, None]
    dy = state["dy"].double()
    dw = (dy * x * r).sum(0)
    g = dy * state["weight"].double()
    c = (g * x).sum(1, keepdim=True) * r / case["d"]
    dx = r * (g - x * r * c)
    return {"dx": dx if state["dsum"] is None else dx + state["dsum"].double(), "dweight": dw}
