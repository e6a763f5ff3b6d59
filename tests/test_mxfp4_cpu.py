"""The 4-bit layer and the rms norm without a GPU: the oracle against closed forms and autograd, arguments and refusals."""

from __future__ import annotations

import ctypes
import itertools

import pytest
import torch

from oracle import mxfp4_block as ob


def _mx():
    import mx_qlinear

    return mx_qlinear


CODES, SCALE = torch.float4_e2m1fn_x2, torch.float8_e8m0fnu


def _codes(m, half):
    return torch.zeros(m, half, dtype=torch.uint8).view(CODES)


def _scale(m, kb):
    return torch.full((m, kb), 127, dtype=torch.uint8).view(SCALE)


# ---------------------------------------------------------------------------------------
# the oracle
# ---------------------------------------------------------------------------------------

def test_rounding_of_ties_and_neighbours():
    ties = {0.25: 0.0, 0.75: 1.0, 1.25: 1.0, 1.75: 2.0, 2.5: 2.0, 3.5: 4.0, 5.0: 4.0}
    t = ob.table()
    for tie, to in ties.items():
        for sign in (1, -1):
            v = torch.tensor([tie, tie * (1 - 2.0**-40), tie * (1 + 2.0**-40)], dtype=torch.float64) * sign
            got = t[ob.round_e2m1(v).long()] * sign
            below = max(x for x in ob.VALUES if x < tie)
            above = min(x for x in ob.VALUES if x > tie)
            assert got.tolist() == [to, below, above]
    assert ob.round_e2m1(ob.table()).tolist() == list(range(16))


def test_exponents_borders():
    for e in (-125, -3, 0, 5, 125):
        top = torch.tensor([6.0 * 2.0**e, 6.0 * 2.0**e * (1 + 2.0**-23), 6.0 * 2.0**e * (1 - 2.0**-24)], dtype=torch.float64)
        assert ob.exponent(top).tolist() == [e, e + 1, e]
    assert ob.exponent(torch.tensor([0.0, 2.0**-140], dtype=torch.float64)).tolist() == [0, -125]


def test_rows_known_block():
    x = torch.zeros(2, 35, dtype=torch.float32)
    x[0, :8] = torch.tensor(ob.VALUES) * 4
    x[0, 34] = -1.0
    x[1, 0] = float("nan")
    v, b, c = ob.rows(x)
    assert b.tolist() == [[129, 125], [255, 127]]
    assert c[0, :8].tolist() == list(range(8)) and c[0, 34] == 14  # -1 = -4 * 2^-2
    assert torch.equal(v[0], x[0].double()) and bool(v[1, :32].isnan().all()) and v[1, 32:].tolist() == [0.0] * 3
    q = ob.pack(c)
    assert q.shape == (2, 18) and torch.equal(ob.unpack(q, 35), c)
    assert torch.equal(ob.values(q, b.to(torch.uint8), 35)[0], x[0].double())


def test_planted_rounding_is_seen():
    """Half up instead of half to even differs on the ties."""
    v = torch.tensor([0.25, 1.25, 2.5, 5.0], dtype=torch.float64)
    up = torch.tensor([0.5, 1.5, 3.0, 6.0], dtype=torch.float64)
    assert not torch.equal(ob.table()[ob.round_e2m1(v).long()], up)


def test_tiles_place_every_byte_once():
    s = torch.arange(70 * 33, dtype=torch.int32).view(70, 33) % 255
    t = ob.tiles(s, 33 * 32)
    assert len(t) == 70 * 33 and max(t) < 3 * 3 * 512


@pytest.mark.parametrize("residual", [False, True])
def test_norm_gradient_is_autograds(residual):
    g = torch.Generator().manual_seed(5)
    x, w = (torch.randn(5, 37, generator=g, dtype=torch.float64, requires_grad=True) for _ in range(2))
    w = torch.randn(37, generator=g, dtype=torch.float64, requires_grad=True)
    dy, ds = torch.randn(5, 37, generator=g, dtype=torch.float64), torch.randn(5, 37, generator=g, dtype=torch.float64)
    rstd = (x.square().mean(1, keepdim=True) + 1e-5).rsqrt()
    y = x * rstd * w
    loss = (y * dy).sum() + ((x * ds).sum() if residual else 0)
    gx, gw = torch.autograd.grad(loss, (x, w))
    dx, dw = ob.rms_norm_backward(dy, x.detach(), rstd.detach().squeeze(1), w.detach(), ds if residual else None)
    assert torch.allclose(dx, gx, rtol=1e-12, atol=1e-12) and torch.allclose(dw, gw, rtol=1e-12, atol=1e-12)


# ---------------------------------------------------------------------------------------
# arguments
# ---------------------------------------------------------------------------------------

def test_functions_refuse_host_tensors():
    mx = _mx()
    x, stat = torch.zeros(4, 256), torch.zeros(4)
    p = mx.PreparedMxfp4Weight(torch.zeros(8, 128, dtype=torch.uint8), torch.zeros(512, dtype=torch.uint8), 8, 256)
    for call in (lambda: mx.quantize_mxfp4(x), lambda: mx.dequantize_mxfp4(_codes(4, 128), _scale(4, 8)),
                 lambda: mx.prepare_mxfp4_weight(x), lambda: mx.prepare_mxfp4_weight(_codes(4, 128), _scale(4, 8)),
                 lambda: mx.mxfp4_linear(x, p), lambda: mx.mxfp4_linear_prequantized(_codes(4, 128), _scale(4, 8), p),
                 lambda: mx.mxfp4_linear_backward(torch.zeros(4, 8), p), lambda: mx.rms_norm(x),
                 lambda: mx.rms_norm_quantize_fp8(x), lambda: mx.rms_norm_quantize_mxfp4(x),
                 lambda: mx.rms_norm_backward(x, x, stat), lambda: mx.Mxfp4Linear(256, 8)(x),
                 lambda: mx.Mxfp4Linear(256, 8)(x.clone().requires_grad_()), lambda: mx.RMSNorm(256)(x)):
        with pytest.raises(RuntimeError, match="GPU only"):
            call()


def test_arguments_are_checked():
    mx = _mx()
    q, s = _codes(4, 128), _scale(4, 8)
    p = mx.PreparedMxfp4Weight(torch.zeros(8, 128, dtype=torch.uint8), torch.zeros(512, dtype=torch.uint8), 8, 256)
    with pytest.raises(ValueError, match="unsupported input dtype"):
        mx.quantize_mxfp4(torch.zeros(4, 256, dtype=torch.int8, device="meta"))
    for bad in (torch.zeros(4), torch.zeros(0, 4)):
        with pytest.raises(ValueError, match="2D"):
            mx.prepare_mxfp4_weight(bad)
    with pytest.raises(ValueError, match="float4_e2m1fn_x2"):
        mx.prepare_mxfp4_weight(torch.zeros(4, 256), s)
    with pytest.raises(ValueError, match="scale of shape"):
        mx.prepare_mxfp4_weight(q, _scale(4, 7))
    with pytest.raises(ValueError, match="width of 254"):
        mx.prepare_mxfp4_weight(q, s, in_features=254)
    with pytest.raises(ValueError, match="in_features"):
        mx.prepare_mxfp4_weight(torch.zeros(4, 256), in_features=255)
    with pytest.raises(TypeError, match="prepare_mxfp4_weight"):
        mx.mxfp4_linear(torch.zeros(4, 256), torch.zeros(4, 256))
    with pytest.raises(TypeError, match="prepare_mxfp4_weight"):
        mx.mxfp4_linear_prequantized(q, s, torch.zeros(4, 256))
    with pytest.raises(TypeError, match="prepare_mxfp4_weight"):
        mx.mxfp4_linear_backward(torch.zeros(4, 8), torch.zeros(8, 256))
    with pytest.raises(ValueError, match="K mismatch"):
        mx.mxfp4_linear(torch.zeros(4, 128), p)
    with pytest.raises(ValueError, match="non-empty"):
        mx.mxfp4_linear(torch.zeros(4, 0), p)
    with pytest.raises(ValueError, match="width of 256"):
        mx.mxfp4_linear_prequantized(_codes(4, 127), s, p)
    with pytest.raises(ValueError, match="scale of shape"):
        mx.mxfp4_linear_prequantized(q, _scale(3, 8), p)
    with pytest.raises(ValueError, match="float8_e8m0fnu"):
        mx.mxfp4_linear_prequantized(q, torch.ones(4, 8), p)
    with pytest.raises(ValueError, match="gradient of shape"):
        mx.mxfp4_linear_backward(torch.zeros(4, 9), p)
    with pytest.raises(ValueError, match="gradient dtype"):
        mx.mxfp4_linear_backward(torch.zeros(4, 8, dtype=torch.int32), p)
    with pytest.raises(ValueError, match="output dtype"):
        mx.mxfp4_linear_backward(torch.zeros(4, 8), p, grad_dtype=torch.int8)
    with pytest.raises(ValueError, match="input features"):
        mx.Mxfp4Linear(128, 8)(torch.zeros(4, 256))
    x, stat = torch.zeros(4, 256), torch.zeros(4)
    for fn in (mx.rms_norm, mx.rms_norm_quantize_fp8, mx.rms_norm_quantize_mxfp4):
        with pytest.raises(ValueError, match="eps"):
            fn(x, eps=-1.0)
        with pytest.raises(ValueError, match="eps"):
            fn(x, eps=float("nan"))
        with pytest.raises(ValueError, match="non-empty"):
            fn(x[:, :0])
        with pytest.raises(ValueError, match="input dtype"):
            fn(x.int())
        with pytest.raises(ValueError, match="residual"):
            fn(x, residual=x.bfloat16())
        with pytest.raises(ValueError, match="residual"):
            fn(x, residual=x[:3])
    with pytest.raises(ValueError, match="input of"):
        mx.rms_norm_backward(x, x.bfloat16(), stat)
    with pytest.raises(ValueError, match="input of shape"):
        mx.rms_norm_backward(x, x[:3], stat)
    with pytest.raises(ValueError, match="input of shape"):
        mx.rms_norm_backward(x, (torch.zeros(4, 128).to(torch.float8_e4m3fn), _scale(4, 1)), stat)
    with pytest.raises(ValueError, match="rstd"):
        mx.rms_norm_backward(x, x, stat.double())
    with pytest.raises(ValueError, match="rstd"):
        mx.rms_norm_backward(x, x, stat[:3])
    with pytest.raises(ValueError, match="gradient of the sum"):
        mx.rms_norm_backward(x, x, stat, dsum=x[:, :8])
    with pytest.raises(ValueError, match="features"):
        mx.RMSNorm(128)(x)


def test_forward_mode_tangents_are_refused():
    mx = _mx()
    from torch.autograd import forward_ad

    with forward_ad.dual_level():
        x = forward_ad.make_dual(torch.zeros(4, 256), torch.ones(4, 256))
        for layer in (mx.RMSNorm(256), mx.Mxfp4Linear(256, 8)):
            with pytest.raises(RuntimeError, match="forward mode"):
                layer(x)
        with pytest.raises(RuntimeError, match="forward mode"):
            mx.RMSNorm(256)(torch.zeros(4, 256), x)


def test_module_buffers():
    """The weight's form is the module's state: buffers, no parameter, kept through casts."""
    mx = _mx()
    layer = mx.Mxfp4Linear(1000, 70, dtype=torch.bfloat16)
    assert [n for n, _ in layer.named_parameters()] == ["bias"]
    state = layer.state_dict()
    assert state["qweight"].shape == (70, 512) and state["scale"].numel() == 3 * 2 * 512
    layer.half()
    assert layer.qweight.dtype == layer.scale.dtype == torch.uint8 and layer.bias.dtype == torch.float16
    other = mx.Mxfp4Linear(1000, 70, dtype=torch.float16)
    other.load_state_dict(layer.state_dict())
    p = other.prepared()
    assert p.q is other.qweight and (p.out_features, p.in_features) == (70, 1000)


def test_storage_in_deterministic_mode():
    """torch fills new tensors in that mode, which it cannot do in the codes' type."""
    from mx_qlinear import mxfp4

    torch.use_deterministic_algorithms(True)
    try:
        q, s = mxfp4._new_pair(3, 130, "cpu")
    finally:
        torch.use_deterministic_algorithms(False)
    for t, want in zip((q, s), mxfp4._new_pair(3, 130, "cpu")):
        assert (t.dtype, t.shape, t.stride()) == (want.dtype, want.shape, want.stride())


# ---------------------------------------------------------------------------------------
# the C entries
# ---------------------------------------------------------------------------------------

def _call(name, *args):
    from mx_qlinear import _lib

    return _lib.call(name, *args, None)


OK = 1 << 20  # an aligned pointer that is never read


def _refused(name, args, places, match=None):
    for i, v in places:
        a = list(args)
        a[i] = v
        with pytest.raises((ValueError, RuntimeError), match=match):
            _call(name, *a)


def test_c_quantizers_refuse_before_any_launch():
    good = [OK, 0, 300, OK, 192, OK, 12, 8, 300]
    _refused("mxq_mxfp4_quantize_rows", good, [(0, None), (1, 3), (2, 299), (3, None), (3, OK + 8), (4, 144), (4, 184), (5, None),
                                               (5, OK + 2), (6, 8), (6, 13), (7, -1), (8, 0), (8, 1 << 30)])
    tiled = [OK, 0, 300, OK, 256, OK, 0, 8, 300]
    _refused("mxq_mxfp4_quantize_rows", tiled, [(4, 192), (4, 240)])
    back = [OK, 150, OK, 10, OK, 0, 8, 300]
    _refused("mxq_mxfp4_dequantize_rows", back, [(0, None), (1, 149), (2, None), (3, 9), (4, None), (5, 5), (6, -1), (7, 0)])
    layout = [OK, 150, OK, 10, OK, 256, OK, 8, 300]
    _refused("mxq_mxfp4_layout", layout, [(0, None), (1, 149), (2, None), (3, 9), (4, OK + 4), (5, 192), (5, 264), (6, None), (7, -1),
                                          (8, 0)])
    _call("mxq_mxfp4_quantize_rows", None, 0, 300, None, 192, None, 12, 0, 300)
    _call("mxq_mxfp4_dequantize_rows", None, 150, None, 10, None, 0, 0, 300)
    _call("mxq_mxfp4_layout", None, 150, None, 10, None, 0, None, 0, 300)


def test_c_products_refuse_before_any_launch():
    from mx_qlinear import _lib

    m, n, k = 40, 100, 300
    gemm = [OK, 256, OK, OK, 256, OK, None, OK, n, 2, m, n, k, None, 0]
    big = [(9, 3), (10, -1), (11, 0), (12, 0), (11, (1 << 22) + 1), (12, (1 << 22) + 1)]
    _refused("mxq_mxfp4_gemm", gemm, [(0, None), (0, OK + 8), (1, 128), (1, 264), (1, 1 << 23), (2, None), (2, OK + 8), (3, None), (3, OK + 4),
                                      (4, 128), (4, 264), (5, None), (5, OK + 8), (7, None), (8, n - 1), *big])
    _call("mxq_mxfp4_gemm", None, 256, None, None, 256, None, None, None, n, 2, 0, n, k, None, 0)
    need = ctypes.c_int64()
    _lib.call("mxq_mxfp4_linear_workspace", m, n, k, ctypes.byref(need))
    assert need.value > 0
    fwd = [OK, 2, k, OK, 256, OK, None, OK, n, 2, m, n, k, OK, need.value]
    _refused("mxq_mxfp4_linear", fwd, [(0, None), (1, 4), (2, k - 1), (3, None), (4, 128), (5, None), (7, None), (8, n - 1), (13, None),
                                       (13, OK + 8), (14, need.value - 1), *big])
    few = [*fwd[:10], 3, n, k, None, 0]
    _refused("mxq_mxfp4_linear", few, [(0, None), (1, 4), (2, k - 1), (3, None), (4, 128), (5, None), (7, None), (8, n - 1), (9, 3)])
    _call("mxq_mxfp4_linear", None, 2, k, None, 256, None, None, None, n, 2, 0, n, k, None, 0)
    _lib.call("mxq_mxfp4_linear_prequantized_workspace", m, n, k, 0, ctypes.byref(need))
    pre = [OK, 150, OK, 10, 0, OK, 256, OK, None, OK, n, 2, m, n, k, OK, need.value]
    _refused("mxq_mxfp4_linear_prequantized", pre, [(0, None), (1, 149), (2, None), (3, 9), (4, 1), (5, None), (6, 128), (7, None), (9, None),
                                                    (10, n - 1), (11, 3), (12, -1), (13, 0), (14, 0), (15, None), (15, OK + 8),
                                                    (16, need.value - 1)])
    few = [*pre[:12], 3, n, k, None, 0]
    _refused("mxq_mxfp4_linear_prequantized", few, [(0, None), (1, 149), (2, None), (3, 9), (5, None), (6, 128), (7, None), (10, n - 1), (11, 3)])
    for dtype, direct, needs in itertools.product((0, 1, 2), (0, 1), (1, 2, 3)):
        _lib.call("mxq_mxfp4_linear_backward_workspace", m, 104, k, dtype, direct if dtype == 2 else 0, needs, ctypes.byref(need))
    _lib.call("mxq_mxfp4_linear_backward_workspace", m, n, k, 0, 0, 3, ctypes.byref(need))
    bwd = [OK, 0, n, 0, OK, 256, OK, OK, OK, 0, m, n, k, OK, need.value]
    _refused("mxq_mxfp4_linear_backward", bwd, [(0, None), (1, 4), (2, n - 1), (3, 1), (4, None), (4, OK + 8), (5, 128), (6, None), (9, 4),
                                                (10, -1), (11, 0), (12, 0), (13, None), (13, OK + 4), (14, need.value - 1)])
    direct = [OK, 2, 104, 1, OK, 256, OK, OK, None, 0, m, 104, k, OK, 1 << 40]
    _refused("mxq_mxfp4_linear_backward", direct, [(0, OK + 8), (1, 1), (2, 108), (2, 1 << 24), (11, 100)])
    for name, args in (("mxq_mxfp4_gemm_workspace", (-1, 8, 8)), ("mxq_mxfp4_linear_workspace", (8, 0, 8)),
                       ("mxq_mxfp4_linear_backward_workspace", (8, 8, 0, 2, 0, 3))):
        with pytest.raises(ValueError):
            _lib.call(name, *args, ctypes.byref(need))


def test_c_norms_refuse_before_any_launch():
    from mx_qlinear import _lib

    d = 300
    same = [OK, OK, 2, d, d, OK, 2, 1e-5, OK, OK, 2, d, None, 0, OK, 4, d]
    _refused("mxq_rms_norm", same, [(0, None), (2, 3), (3, d - 1), (4, d - 1), (6, 5), (7, -1.0), (7, float("nan")), (8, None), (9, None),
                                    (10, 0), (10, 3), (15, -1), (16, 0), (16, 24577)])
    fp8 = [*same[:10], 5, 384, OK, 4, *same[14:]]
    _refused("mxq_rms_norm", fp8, [(9, OK + 4), (11, 256), (11, 388), (12, None), (13, 2)])
    fp4 = [*same[:10], 8, 192, OK, 12, *same[14:]]
    _refused("mxq_rms_norm", fp4, [(9, OK + 2), (11, 150), (11, 194), (12, None), (12, OK + 2), (13, 10), (13, 14)])
    _call("mxq_rms_norm", None, None, 2, d, d, None, 2, 1e-5, None, None, 2, d, None, 0, None, 0, d)
    need = ctypes.c_int64()
    _lib.call("mxq_rms_norm_backward_workspace", 4, d, ctypes.byref(need))
    back = [OK, 2, d, OK, 2, d, None, 0, OK, OK, 2, OK, d, OK, OK, 4, d, OK, need.value]
    _refused("mxq_rms_norm_backward", back, [(0, None), (1, 3), (2, d - 1), (3, None), (4, 0), (4, 5), (5, d - 1), (8, None), (10, 3), (12, d - 1),
                                             (13, None), (15, -1), (16, 0), (16, 24577), (17, None), (18, need.value - 4)])
