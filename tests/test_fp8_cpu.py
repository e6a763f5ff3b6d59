"""8-bit floating point layer without a GPU: the oracle's closed forms and the refusals, on the host before any launch."""

from __future__ import annotations

import ctypes

import pytest
import torch

from oracle import fp8_block as ob


def _mx():
    import mx_qlinear

    return mx_qlinear


def test_oracle_rounding_is_torchs():
    v = torch.cat([torch.linspace(-448, 448, 20001, dtype=torch.float64), torch.linspace(-0.1, 0.1, 20001, dtype=torch.float64)])
    v = v.float().double()
    assert torch.equal(ob.round_e4m3(v), v.float().to(torch.float8_e4m3fn).double())
    t = ob.e4m3_table()
    codes = torch.arange(256).to(torch.uint8).view(torch.float8_e4m3fn).double()
    assert torch.equal(t.nan_to_num(1e9), codes.nan_to_num(1e9))


def test_oracle_exponents():
    a = torch.tensor([0.0, 448.0, 448.0000001, 224.0, 2.0**-108, 448 * 2.0**-117, 2.0**-149, 3.4e38], dtype=torch.float64)
    e = ob.exponent(a)
    assert e.tolist() == [0, 0, 1, -1, -116, -117, -117, 120]
    s = torch.ldexp(torch.ones((), dtype=torch.float64), e)
    assert bool((a <= 448 * s).all())


def test_oracle_layer_norm_is_autograds():
    g = torch.Generator().manual_seed(4)
    x, w, b, dy = (torch.randn(n, 37, generator=g, dtype=torch.float64) for n in (6, 1, 1, 6))
    w, b = w[0], b[0]
    xs = [t.clone().requires_grad_() for t in (x, w, b)]
    y = torch.nn.functional.layer_norm(xs[0], (37,), xs[1], xs[2], 1e-5)
    y.backward(dy)
    got, mean, rstd = ob.layer_norm(x, w, b, 1e-5)
    torch.testing.assert_close(got, y.detach(), rtol=1e-12, atol=1e-12)
    for a, t in zip(ob.layer_norm_backward(dy, x, mean, rstd, w), xs):
        torch.testing.assert_close(a, t.grad, rtol=1e-11, atol=1e-11)


def test_cpu_tensors_are_refused():
    mx = _mx()
    x = torch.zeros(4, 256)
    with pytest.raises(RuntimeError, match="GPU only"):
        mx.quantize_fp8_block128(x)
    with pytest.raises(RuntimeError, match="GPU only"):
        mx.prepare_fp8_weight(x)
    q, s = x.to(torch.float8_e4m3fn), torch.ones(4, 2).to(torch.float8_e8m0fnu)
    with pytest.raises(RuntimeError, match="GPU only"):
        mx.dequantize_fp8_block128(q, s)
    with pytest.raises(RuntimeError, match="GPU only"):
        mx.prepare_fp8_weight(torch.zeros(128, 256).to(torch.float8_e4m3fn), torch.ones(1, 2).to(torch.float8_e8m0fnu))


def test_arguments_are_checked():
    mx = _mx()
    q, s = torch.zeros(4, 256).to(torch.float8_e4m3fn), torch.ones(4, 2).to(torch.float8_e8m0fnu)
    p = mx.PreparedFp8Weight(q, s, None, None, 4, 256)
    with pytest.raises(ValueError, match="unsupported input dtype"):
        mx.quantize_fp8_block128(torch.zeros(4, 256, dtype=torch.int8, device="meta"))
    with pytest.raises(ValueError, match="2D"):
        mx.prepare_fp8_weight(torch.zeros(4))
    with pytest.raises(ValueError, match="2D"):
        mx.prepare_fp8_weight(torch.zeros(0, 4))
    with pytest.raises(ValueError, match="scale of shape"):
        mx.prepare_fp8_weight(torch.zeros(300, 256).to(torch.float8_e4m3fn), s)
    with pytest.raises(ValueError, match="float8_e4m3fn"):
        mx.prepare_fp8_weight(torch.zeros(4, 256), s)
    with pytest.raises(TypeError, match="prepare_fp8_weight"):
        mx.fp8_linear(torch.zeros(4, 256), torch.zeros(4, 256))
    with pytest.raises(ValueError, match="K mismatch"):
        mx.fp8_linear(torch.zeros(4, 128), p)
    with pytest.raises(ValueError, match="non-empty"):
        mx.fp8_linear(torch.zeros(4, 0), p)
    with pytest.raises(ValueError, match="scale of shape"):
        mx.fp8_linear_prequantized(q, torch.ones(4, 3).to(torch.float8_e8m0fnu), p)
    with pytest.raises(ValueError, match="float8_e4m3fn"):
        mx.fp8_linear_prequantized(q, torch.ones(4, 2), p)


def _call(name, *args):
    from mx_qlinear import _lib

    return _lib.call(name, *args, None)


def test_c_entries_refuse_before_any_launch():
    """Sizes, strides, dtypes, pointers and workspaces (16 stands for an aligned pointer that is never read)."""
    ok = 1 << 20
    with pytest.raises(ValueError, match="dtype"):
        _call("mxq_fp8_quantize_rows", ok, 3, 256, ok, 256, ok, 4, 8, 256)
    for ldx, ldq, lds, k in ((255, 256, 4, 256), (256, 128, 4, 256), (256, 264, 4, 256), (256, 256, 1, 256), (256, 256, 4, 0)):
        with pytest.raises(ValueError):
            _call("mxq_fp8_quantize_rows", ok, 0, ldx, ok, ldq, ok, lds, 8, k)
    with pytest.raises(ValueError, match="misaligned"):
        _call("mxq_fp8_quantize_rows", ok, 0, 256, ok + 8, 256, ok, 4, 8, 256)
    with pytest.raises(ValueError, match="null"):
        _call("mxq_fp8_dequantize_rows", None, 256, ok, 2, ok, 0, 8, 256)
    with pytest.raises(ValueError):
        _call("mxq_fp8_quantize_tiles", ok, 0, 256, ok, 256, ok, 4, ok, 128, ok, 0, 8, 256)
    with pytest.raises(ValueError, match="activations"):
        _call("mxq_fp8_gemm", ok, 200, ok, 4, ok, 256, ok, 4, None, ok, 128, 2, 100, 128, 256, None, 0)
    with pytest.raises(ValueError, match="weight"):
        _call("mxq_fp8_gemm", ok, 256, ok, 4, ok, 256, ok, 2, None, ok, 128, 2, 100, 128, 256, None, 0)
    with pytest.raises(ValueError, match="weight"):
        _call("mxq_fp8_gemm", ok, 256, ok, 4, ok, 256, ok, 4, None, ok, 127, 2, 100, 128, 256, None, 0)
    with pytest.raises(ValueError, match="misaligned"):
        _call("mxq_fp8_gemm", ok + 1, 256, ok, 4, ok, 256, ok, 4, None, ok, 128, 2, 100, 128, 256, None, 0)
    need = ctypes.c_int64()
    from mx_qlinear import _lib

    _lib.call("mxq_fp8_gemm_workspace", 128, 256, 16384, ctypes.byref(need))
    assert need.value > 0  # two tiles: K is split
    with pytest.raises(ValueError, match="workspace"):
        _call("mxq_fp8_gemm", ok, 16384, ok, 128, ok, 16384, ok, 128, None, ok, 256, 2, 128, 256, 16384, ok, need.value - 16)
    with pytest.raises(ValueError, match="activations"):
        _call("mxq_fp8_linear", ok, 2, 249, ok, 256, ok, 4, None, ok, 128, 2, 4, 128, 250, None, 0)
    with pytest.raises(ValueError):
        _call("mxq_fp8_grad_pass", ok, 2, 256, ok, 256, ok, 4, ok, 2, 256, None, 0, 8, 256)
    # no rows: nothing to do, no pointer needed
    _call("mxq_fp8_quantize_rows", None, 0, 256, None, 256, None, 4, 0, 256)
    _call("mxq_fp8_gemm", None, 256, None, 4, None, 256, None, 4, None, None, 128, 2, 0, 128, 256, None, 0)


def test_gradient_arguments_are_checked():
    mx = _mx()
    q, s = torch.zeros(4, 256).to(torch.float8_e4m3fn), torch.ones(4, 2).to(torch.float8_e8m0fnu)
    p = mx.PreparedFp8Weight(q, s, None, None, 8, 256)
    with pytest.raises(ValueError, match="transposed"):
        mx.fp8_linear_backward(torch.zeros(4, 8), q, s, p)
    with pytest.raises(ValueError, match="gradient of shape"):
        mx.fp8_linear_backward(torch.zeros(4, 9), q, s, p)
    with pytest.raises(ValueError, match="gradient dtype"):
        mx.fp8_linear_backward(torch.zeros(4, 8, dtype=torch.int32), q, s, p)
    with pytest.raises(ValueError, match="output dtype"):
        mx.fp8_linear_backward(torch.zeros(4, 8), q, s, p, grad_dtype=torch.int8)
    with pytest.raises(RuntimeError, match="GPU only"):
        mx.fp8_linear_backward(torch.zeros(4, 8), q, s, p, (False, True, True))
    x, stat = torch.zeros(4, 256), torch.zeros(4)
    with pytest.raises(RuntimeError, match="GPU only"):
        mx.layer_norm(x)
    with pytest.raises(ValueError, match="eps"):
        mx.layer_norm(x, eps=-1.0)
    with pytest.raises(ValueError, match="non-empty"):
        mx.layer_norm(x[:, :0])
    with pytest.raises(ValueError, match="input dtype"):
        mx.layer_norm(x.int())
    with pytest.raises(ValueError, match="input of"):
        mx.layer_norm_backward(x, x.bfloat16(), stat, stat)
    with pytest.raises(ValueError, match="input of shape"):
        mx.layer_norm_backward(x, (q[:, :128], s[:, :1]), stat, stat)
    with pytest.raises(ValueError, match="mean"):
        mx.layer_norm_backward(x, x, stat[:3], stat)
    with pytest.raises(ValueError, match="rstd"):
        mx.layer_norm_backward(x, x, stat, stat.double())
    with pytest.raises(ValueError, match="input features"):
        mx.Fp8Linear(128, 8)(x)
    with pytest.raises(ValueError, match="features"):
        mx.LayerNorm(128)(x)


def test_c_gradient_entries_refuse_before_any_launch():
    from mx_qlinear import _lib

    ok = 1 << 20
    for args in ((ok, 0, 256, ok, 256, ok, 2, ok, 0, 8, 256, 256), (ok, 1, 250, ok, 256, ok, 2, ok, 0, 8, 250, 256),
                 (ok, 1, 256, ok, 248, ok, 2, ok, 0, 8, 256, 248), (ok, 1, 256, ok, 256, ok, 1, ok, 0, 8, 256, 256),
                 (ok + 2, 1, 256, ok, 256, ok, 2, ok, 0, 8, 256, 256), (ok, 1, 256, ok, 256, ok, 2, ok, 5, 8, 256, 256)):
        with pytest.raises(ValueError):
            _call("mxq_fp8_wgrad", *args, None, 0)
    need = ctypes.c_int64()
    _lib.call("mxq_fp8_wgrad_workspace", 65536, 256, 256, 1, ctypes.byref(need))
    assert need.value > 0
    with pytest.raises(ValueError, match="workspace"):
        _call("mxq_fp8_wgrad", ok, 1, 256, ok, 256, ok, 2, ok, 0, 65536, 256, 256, None, 0)
    with pytest.raises(_lib.MxqError, match="24576"):
        _call("mxq_layer_norm", ok, 2, 24577, None, None, 2, 1e-5, ok, None, None, 4, 24577)
    with pytest.raises(ValueError):
        _call("mxq_layer_norm", ok, 2, 127, None, None, 2, 1e-5, ok, None, None, 4, 128)
    with pytest.raises(ValueError, match="workspace"):
        _call("mxq_layer_norm_backward", ok, 2, 128, ok, 2, 128, None, 0, ok, ok, None, 2, ok, ok, 4, 128, ok, 8)
    with pytest.raises(ValueError, match="dtype code"):
        _call("mxq_layer_norm_backward", ok, 2, 128, ok, 0, 128, None, 0, ok, ok, None, 2, ok, None, 4, 128, None, 0)
    with pytest.raises(ValueError, match="null"):
        _call("mxq_layer_norm_backward", ok, 2, 128, ok, 5, 128, None, 1, ok, ok, None, 2, ok, None, 4, 128, None, 0)
    with pytest.raises(ValueError, match="directly"):
        _call("mxq_fp8_linear_backward", ok, 1, 256, 1, ok, 256, ok, 2, 1, ok, 256, ok, 4, ok, ok, ok, 0, 8, 256, 256, ok, 1 << 30)
    with pytest.raises(ValueError, match="workspace"):
        _call("mxq_fp8_linear_backward", ok, 1, 256, 0, ok, 256, ok, 2, 1, ok, 256, ok, 4, ok, ok, ok, 0, 8, 256, 256, None, 0)
    with pytest.raises(ValueError, match="workspace"):
        _call("mxq_fp8_linear", ok, 2, 256, ok, 256, ok, 4, None, ok, 128, 2, 100, 128, 256, ok, 64)
    with pytest.raises(ValueError, match="size"):
        _call("mxq_fp8_linear", ok, 2, 256, ok, 256, ok, 4, None, ok, 128, 2, 100, 0, 256, ok, 64)
    with pytest.raises(ValueError, match="strides"):
        _call("mxq_fp8_prepare_tiles", ok, 99, ok, 1, ok, 128, ok, 4, None, 0, None, 0, 100, 100)
    with pytest.raises(ValueError, match="scale"):
        _call("mxq_fp8_prepare_tiles", ok, 300, ok, 2, ok, 384, ok, 4, None, 0, None, 0, 100, 300)
    with pytest.raises(ValueError, match="strides"):
        _call("mxq_pad_rows", ok, 100, 100, ok, 104, 4)


def test_whole_passes_refuse_before_their_first_launch():
    """Strides and pointers that only a later step of the pass reads (a launch would fail here with another error)."""
    ok, room = 1 << 20, 1 << 34

    def forward(ldb=256, sb=ok, ldsb=4, d=ok, ldd=128, b=ok, bias=None, out=2):
        _call("mxq_fp8_linear", ok, 2, 256, b, ldb, sb, ldsb, bias, d, ldd, out, 100, 128, 256, ok, room)

    for bad in ({"ldb": 128}, {"ldb": 264}, {"sb": None}, {"sb": ok + 1}, {"ldsb": 2}, {"d": None}, {"ldd": 100}, {"b": ok + 4}, {"out": 9}):
        with pytest.raises(ValueError):
            forward(**bad)

    def backward(q=ok, ldq=256, scale=ok, lds=2, readable=1, bt=ok, ldbt=128, sbt=ok, ldsbt=4, dy=ok, ldy=128, direct=0, m=100):
        _call("mxq_fp8_linear_backward", dy, 2, ldy, direct, q, ldq, scale, lds, readable, bt, ldbt, sbt, ldsbt, ok, ok, ok, 0, m, 128,
              256, ok, room)

    for bad in ({"q": None}, {"q": ok + 8}, {"ldq": 128}, {"ldq": 264}, {"ldq": 1 << 24}, {"scale": None}, {"lds": 1}, {"bt": None},
                {"bt": ok + 8}, {"ldbt": 64}, {"sbt": None}, {"ldsbt": 1}, {"sbt": ok + 2}, {"readable": 0, "ldq": 128},
                {"readable": 0, "q": None}, {"dy": None}, {"ldy": 127}, {"direct": 1, "ldy": 1 << 24}):
        with pytest.raises(ValueError):
            backward(**bad)


def test_full_sums_take_the_same_workspace():
    from mx_qlinear import _lib

    plain, full = ctypes.c_int64(), ctypes.c_int64()
    for needs in range(1, 8):
        _lib.call("mxq_fp8_linear_backward_workspace", 700, 300, 500, 1, 0, 1, needs, ctypes.byref(plain))
        _lib.call("mxq_fp8_linear_backward_workspace", 700, 300, 500, 1 | _lib.FP8_FULL_SUMS, 0, 1, needs, ctypes.byref(full))
        assert plain.value == full.value
    with pytest.raises(ValueError):
        _lib.call("mxq_fp8_linear_backward_workspace", 700, 300, 500, 3 | _lib.FP8_FULL_SUMS, 0, 1, 7, ctypes.byref(full))
