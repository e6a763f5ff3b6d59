"""Every kernel form of the 4-bit layer at sizes that take it: workgroups of one to six blocks of sixteen weight rows in four and
eight waves, the product's three tiles and the input's gradient's three, whole and in slices, with odd and even numbers of
stages and edges that no tile divides.

The plans say which form a size takes (256 CUs), so a later change of their costs cannot leave a form untested. Operands are
held to the definition: codes and scales are random bytes whose values are a table's, and both sides' products are taken in
float64 on the card. Bounds are those of test_gpu_mxfp4.py; the gradient's as a norm is one rounding of 2^-24 of the result per
addend, of independent sign.
"""

from __future__ import annotations

import math

import pytest
import torch

from oracle import mxfp4_block as ob

CODES, SCALE = torch.float4_e2m1fn_x2, torch.float8_e8m0fnu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
DTYPES = [BF16, F16, F32]
TYPE_CODE = {F32: 0, F16: 1, BF16: 2}
PARTS = {BF16: 1, F16: 2, F32: 3}

# (M, N, K): weight rows and waves of a workgroup
FEW_ROWS = {
    (1, 20480, 5120): (16, 4), (15, 33, 4100): (12, 8),
    (1, 4099, 5120): (20, 4), (16, 13001, 1030): (28, 4), (1, 5120, 20480): (20, 8),
    (7, 9001, 1030): (36, 4), (3, 21501, 1030): (44, 4), (4, 21504, 5376): (44, 4), (16, 8900, 1922): (36, 8),
    (15, 12700, 2300): (52, 8), (16, 30001, 2500): (60, 8),
    (16, 18001, 3000): (72, 8), (16, 20480, 5120): (80, 8),
    (16, 20483, 5000): (84, 8), (16, 21504, 5376): (84, 8), (12, 24001, 5376): (96, 8),
}
# (M, N, K): tile and K slices
PRODUCTS = {
    (900, 2049, 20001): ((128, 128), 1), (700, 5000, 2200): ((128, 128), 1), (700, 2049, 19700): ((128, 128), 2),
    (200, 5120, 20480): ((128, 128), 3), (130, 1000, 9000): ((128, 128), 9),
    (515, 9001, 777): ((128, 256), 1), (1300, 3001, 2049): ((128, 256), 1), (1100, 5000, 1000): ((128, 256), 1),
    (2049, 1030, 40960): ((128, 256), 3),
    (1025, 20481, 512): ((256, 256), 1), (1030, 9001, 777): ((256, 256), 1), (1030, 9001, 2049): ((256, 256), 1),
    (1030, 9001, 4100): ((256, 256), 1), (2000, 4099, 8191): ((256, 256), 1),
    (1030, 5120, 40960): ((256, 256), 2), (8766, 133, 23929): ((256, 256), 6),
}
# (M, N, K): tile and N slices of gradients in one, two and three parts
GRADIENTS = {
    (515, 2000, 9001): [((128, 128), 1)] * 3, (300, 5000, 4097): [((128, 128), 5)] * 3,
    (1, 1030, 9001): [((64, 256), 9)] * 3, (33, 1030, 9001): [((128, 128), 6), ((64, 256), 9), ((64, 256), 9)],
    (64, 3001, 12300): [((64, 256), 8)] * 3, (50, 5000, 9001): [((64, 256), 14)] * 3, (40, 20480, 5120): [((64, 256), 25)] * 3,
    (1030, 300, 9001): [((256, 256), 1)] * 3, (1030, 1030, 9001): [((256, 256), 1)] * 3, (2050, 777, 5001): [((256, 256), 1)] * 3,
    (130, 2964, 6641): [((128, 128), 4), ((256, 256), 8), ((256, 256), 8)],
    (700, 3001, 5120): [((128, 128), 1), ((128, 128), 2), ((256, 256), 4)], (700, 20480, 5120): [((256, 256), 4)] * 3,
}


def _mx():
    import mx_qlinear

    return mx_qlinear


def _lib():
    from mx_qlinear import _lib

    if not _lib.LIB_PATH.exists():
        from mx_qlinear import build

        build.build()
    return _lib


# ---------------------------------------------------------------------------------------
# the plans
# ---------------------------------------------------------------------------------------

def test_sizes_take_their_forms():
    lib = _lib()
    for (m, n, k), form in FEW_ROWS.items():
        for pair in (False, True):
            plan = lib.mxfp4_plan(m, n, k, pair)
            assert ((plan["rows"], plan["waves"]), plan["tile"], plan["slices"]) == (form, (0, 0), 0), (m, n, k)
    for (m, n, k), form in PRODUCTS.items():
        for pair in (False, True):
            plan = lib.mxfp4_plan(m, n, k, pair)
            assert (plan["rows"], plan["waves"]) == (0, 0) and (plan["tile"], plan["slices"]) == form, (m, n, k)
    for (m, n, k), forms in GRADIENTS.items():
        for dtype in DTYPES:
            plan = lib.mxfp4_backward_plan(m, n, k, TYPE_CODE[dtype])
            assert (plan["tile"], plan["slices"]) == forms[PARTS[dtype] - 1], (m, n, k, dtype)


def test_no_form_is_missing():
    """What the kernels are built for."""
    assert {((rows + 15) // 16, waves) for rows, waves in FEW_ROWS.values()} == (
        {(b, 4) for b in (1, 2, 3)} | {(b, 8) for b in (1, 2, 3, 4, 5, 6)})
    tiles = {(tile, slices > 1) for tile, slices in PRODUCTS.values()}
    assert tiles == {(t, s) for t in ((128, 128), (128, 256), (256, 256)) for s in (False, True)}
    for tile, _ in tiles:  # whole stages of 256 columns (512 of the smallest tile), odd and even
        step = 512 if tile == (128, 128) else 256
        assert {-(-k // step) % 2 for (_, _, k), (t, _) in PRODUCTS.items() if t == tile} == {0, 1}
    for part in range(3):
        forms = {(tile, slices > 1) for f in GRADIENTS.values() for tile, slices in f[part:part + 1]}
        assert forms == {((128, 128), False), ((128, 128), True), ((64, 256), True), ((256, 256), False), ((256, 256), True)}


def test_plans_refuse_bad_sizes():
    lib = _lib()
    for bad in ((0, 8, 8), (-1, 8, 8), (8, 0, 8), (8, 8, 0), (8, (1 << 22) + 1, 8), (8, 8, (1 << 22) + 1)):
        with pytest.raises(ValueError):
            lib.mxfp4_plan(*bad)
        with pytest.raises(ValueError):
            lib.mxfp4_backward_plan(*bad, 2)
    with pytest.raises(ValueError):
        lib.mxfp4_backward_plan(8, 8, 8, 5)
    with pytest.raises(ValueError):
        lib.call("mxq_mxfp4_linear_plan", 8, 8, 8, 0, None)


# ---------------------------------------------------------------------------------------
# on the card
# ---------------------------------------------------------------------------------------

def _values(q, s, k):
    """float64 values of code bytes [rows, ceil(k / 2)] and scale bytes [rows, ceil(k / 32)] where they are."""
    v = ob.table().to(q.device)[torch.stack((q & 15, q >> 4), -1).view(q.shape[0], -1)[:, :k].long()]
    e = torch.ldexp(torch.ones((), dtype=torch.float64, device=q.device), s.int() - 127)
    return v * torch.where(s == 255, math.nan, e).repeat_interleave(32, 1)[:, :k]


def _weight(dev, n, k, seed):
    """(codes, scales) bytes of a weight: every code, scales within 2^12 of each other."""
    g = torch.Generator(device=dev).manual_seed(seed)
    q = torch.randint(0, 256, (n, -(-k // 2)), generator=g, device=dev, dtype=torch.uint8)
    return q, torch.randint(116, 129, (n, -(-k // 32)), generator=g, device=dev, dtype=torch.uint8)


def _rows(dev, m, k, dtype, seed):
    g = torch.Generator(device=dev).manual_seed(seed)
    return (torch.randn(m, k, generator=g, device=dev) * torch.exp(torch.randn(m, 1, generator=g, device=dev))).to(dtype)


def _prepare(q, s, k):
    return _mx().prepare_mxfp4_weight(q.view(CODES), s.view(SCALE), in_features=k)


def check(got, ref, bound, norm):
    u = torch.finfo(got.dtype).eps / 2
    err = (got.double() - ref).abs()
    bound = (bound + u * ref.abs() + torch.finfo(got.dtype).tiny) * (1 + u)
    assert got.shape == ref.shape
    bad = ~(err <= bound)
    assert not bool(bad.any()), (f"{int(bad.sum())} off, the first at {bad.nonzero()[0].tolist()}, worst "
                                 f"{float((err / bound).nan_to_num(math.inf).max())} of the bound")
    assert float(err.norm() / ref.norm()) <= u + norm


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k", [*FEW_ROWS, *PRODUCTS])
def test_products(dev, dtype, m, n, k):
    mx, lib = _mx(), _lib()
    plan = lib.mxfp4_plan(m, n, k)
    assert ((plan["rows"], plan["waves"]) if m <= 16 else (plan["tile"], plan["slices"])) == {**FEW_ROWS, **PRODUCTS}[m, n, k]
    q, s = _weight(dev, n, k, m + n + k)
    weight, wv = _prepare(q, s, k), _values(q, s, k)
    x = _rows(dev, m, k, dtype, n + k)
    bias = _rows(dev, 1, n, dtype, m)[0] if (m + n + k) % 2 else None
    xq, xs = mx.quantize_mxfp4(x)
    xv = _values(xq.view(torch.uint8), xs.view(torch.uint8), k)
    ref = xv @ wv.t()
    cuts = -(-k // 64) * 5 * 2.0**-22
    bound = 2 * cuts * (xv.abs() @ wv.abs().t())
    if bias is not None:
        ref += bias.double()
        bound += 2.0**-23 * (ref.abs() + bias.double().abs())
    y = mx.mxfp4_linear(x, weight, bias)
    assert y.dtype == dtype
    check(y, ref, bound, cuts / 2 + 2.0**-23)
    z = mx.mxfp4_linear_prequantized(xq, xs, weight, bias, dtype)
    check(z, ref, bound, cuts / 2 + 2.0**-23)
    if m > 16:
        assert torch.equal(y, z)
    # a pair at odd places, whose codes are copied
    far = torch.zeros(m, xq.shape[1] + 3, dtype=torch.uint8, device=dev)
    far[:, 1:1 + xq.shape[1]] = xq.view(torch.uint8)
    assert torch.equal(mx.mxfp4_linear_prequantized(far[:, 1:1 + xq.shape[1]].view(CODES), xs, weight, bias, dtype), z)
    assert torch.equal(mx.mxfp4_linear(x, weight, bias), y)  # (the same bits on every run)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k", [*GRADIENTS])
def test_gradients(dev, dtype, m, n, k):
    mx, lib = _mx(), _lib()
    plan = lib.mxfp4_backward_plan(m, n, k, TYPE_CODE[dtype])
    assert (plan["tile"], plan["slices"]) == GRADIENTS[m, n, k][PARTS[dtype] - 1]
    q, s = _weight(dev, n, k, m + n + k)
    weight, wv = _prepare(q, s, k), _values(q, s, k)
    dy = (_rows(dev, m, n, F32, n + k) * 1e-2).to(dtype)
    dyd = dy.double()
    dx, db = mx.mxfp4_linear_backward(dy, weight)
    assert dx.dtype == dtype and db.dtype == F32
    check(dx, dyd @ wv, 2.0**-24 * (PARTS[dtype] * n + 2) * (dyd.abs() @ wv.abs()), 2.0**-24 * math.sqrt(PARTS[dtype] * n))
    check(db[None], dyd.sum(0, keepdim=True), 2.0**-24 * (m + 2) * dyd.abs().sum(0, keepdim=True), 2.0**-24 * math.sqrt(m))
    again, none = mx.mxfp4_linear_backward(dy, weight, (True, False))
    assert none is None and torch.equal(again, dx)


def test_a_wrong_block_is_seen():
    """The table's values are the oracle's; one scale byte of a row's largest block off by one is beyond the bounds."""
    host = torch.device("cpu")
    q, s = _weight(host, 40, 1003, 1)
    wv = _values(q, s, 1003)
    assert torch.equal(wv, ob.values(q, s, 1003))
    xv = _rows(host, 20, 1003, BF16, 2).double()
    ref, cuts = xv @ wv.t(), 16 * 5 * 2.0**-22
    bound = 2 * cuts * (xv.abs() @ wv.abs().t())
    check(ref.float(), ref, bound, cuts / 2)
    s[39, s[39].argmax()] += 1
    with pytest.raises(AssertionError, match="off, the first at"):
        check((xv @ _values(q, s, 1003).t()).float(), ref, bound, cuts / 2)


SPREAD = [(16, 13001, 1030), (16, 20483, 5000), (515, 9001, 777), (1030, 9001, 2049), (200, 5120, 20480), (2049, 1030, 40960)]


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", SPREAD)
def test_nan_stays_in_its_rows_and_columns(dev, m, n, k):
    mx = _mx()
    (q, s), x = _weight(dev, n, k, 1), _rows(dev, m, k, BF16, 2)
    clean = mx.mxfp4_linear(x, _prepare(q, s, k))
    rows, cols = [0, m // 2, m - 1], [0, 33, n // 2, n - 1]
    for i, r in enumerate(rows):
        x[r, (0, k // 2, k - 1)[i]] = math.nan
    for i, c in enumerate(cols):
        s[c, (0, 5, s.shape[1] // 2, s.shape[1] - 1)[i]] = 255
    y = mx.mxfp4_linear(x, _prepare(q, s, k))
    bad = torch.zeros(m, n, dtype=torch.bool, device=dev)
    bad[rows], bad[:, cols] = True, True
    assert bool(y[bad].isnan().all()) and torch.equal(y[~bad], clean[~bad])


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(64, 3001, 12300), (1030, 300, 9001), (700, 20480, 5120)])
def test_nan_in_the_gradient_stays_in_its_rows_and_columns(dev, m, n, k):
    mx = _mx()
    (q, s), dy = _weight(dev, n, k, 1), _rows(dev, m, n, BF16, 2)
    clean = mx.mxfp4_linear_backward(dy, _prepare(q, s, k))[0]
    dy[0, n - 1], dy[m - 1, 0] = math.nan, math.nan
    s[n - 1, 3], s[0, s.shape[1] - 1] = 255, 255
    dx = mx.mxfp4_linear_backward(dy, _prepare(q, s, k))[0]
    bad = torch.zeros(m, k, dtype=torch.bool, device=dev)
    bad[0], bad[m - 1], bad[:, 96:128], bad[:, (s.shape[1] - 1) * 32:] = True, True, True, True
    assert bool(dx[bad].isnan().all()) and torch.equal(dx[~bad], clean[~bad])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k", SPREAD)
def test_nothing_is_written_behind_the_rows(dev, dtype, m, n, k):
    """Results into rows with seven elements behind them, and with others in front and behind."""
    import ctypes

    from mx_qlinear.ops import _launch

    mx, lib = _mx(), _lib()
    q, s = _weight(dev, n, k, 1)
    weight, x = _prepare(q, s, k), _rows(dev, m, k, dtype, 2)
    want = mx.mxfp4_linear(x, weight)
    code, out = TYPE_CODE[dtype], torch.full((m + 2, n + 7), 7.0, dtype=dtype, device=dev)
    need = ctypes.c_int64()
    with torch.cuda.device(dev):
        lib.call("mxq_mxfp4_linear_workspace", m, n, k, ctypes.byref(need))
    ws = torch.empty(need.value, dtype=torch.uint8, device=dev)
    _launch(dev, "mxq_mxfp4_linear", x.data_ptr(), code, k, weight.q.data_ptr(), weight.q.shape[1], weight.scale.data_ptr(), None,
            out[1:].data_ptr(), n + 7, code, m, n, k, ws.data_ptr() if need.value else None, need.value)
    assert torch.equal(out[1:m + 1, :n], want)
    out[1:m + 1, :n] = 7.0
    assert bool((out == 7.0).all())


def _far(dev, t, stride, offset=0):
    """``t [rows, cols]`` as rows ``stride`` elements apart, ``offset`` from the start of their memory."""
    raw = t.view(torch.uint8) if t.dtype in (CODES, SCALE) else t
    base = torch.empty((t.shape[0] - 1) * stride + t.shape[1] + offset, dtype=raw.dtype, device=dev)
    far = base.as_strided(t.shape, (stride, 1), offset)
    far.copy_(raw)
    return far.view(t.dtype) if t.dtype in (CODES, SCALE) else far


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 7, 16, 40, 300])
@pytest.mark.parametrize("stride", [(1 << 22) - 16, 1 << 22, (1 << 22) + 16, (1 << 24) + 3])
def test_rows_far_apart(dev, m, stride):
    """Inputs and pairs whose rows are at and beyond the strides that the products read in place: the same bits as of contiguous
    rows."""
    mx = _mx()
    n, k = 520, 1024
    weight = _prepare(*_weight(dev, n, k, 1), k)
    x = _rows(dev, m, k, BF16, 2)
    pair = mx.quantize_mxfp4(x)
    far = _far(dev, x, stride)
    assert torch.equal(mx.mxfp4_linear(far, weight), mx.mxfp4_linear(x, weight))
    for a, b in zip(mx.quantize_mxfp4(far), pair):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    want = mx.mxfp4_linear_prequantized(*pair, weight)
    for off in (0, 5):
        q, s = _far(dev, pair[0], stride, off), _far(dev, pair[1], stride, off)
        assert torch.equal(mx.mxfp4_linear_prequantized(q, s, weight), want)
        assert torch.equal(mx.dequantize_mxfp4(q, s), mx.dequantize_mxfp4(*pair))
    w, r = _rows(dev, 1, k, BF16, 3)[0], _far(dev, _rows(dev, m, k, BF16, 4), stride, 1)
    y, total, rstd = mx.rms_norm(far, w, residual=r, return_rstd=True)
    for a, b in zip((y, total, rstd), mx.rms_norm(x, w, residual=r.contiguous(), return_rstd=True)):
        assert torch.equal(a, b)
    kept = mx.quantize_fp8_block128(x)
    q8 = torch.empty((m - 1) * stride + k, dtype=torch.float8_e4m3fn, device=dev).as_strided((m, k), (stride, 1)).copy_(kept[0])
    for x_far, x_near in ((far, x), ((q8, kept[1]), kept)):
        for a, b in zip(mx.rms_norm_backward(r, x_far, rstd, w, far), mx.rms_norm_backward(r.contiguous(), x_near, rstd, w, x)):
            assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("m,n,k", [(40, 1032, 20001), (70, 520, 300), (130, 64, 40001)])
def test_gradient_rows_far_apart(dev, dtype, m, n, k):
    """Up to the largest stride that is read in place (2^24 - 8), at it and beyond, in each of the tiles."""
    mx = _mx()
    weight = _prepare(*_weight(dev, n, k, 1), k)
    dy = _rows(dev, m, n, dtype, 2)
    want = mx.mxfp4_linear_backward(dy, weight)
    for stride in ((1 << 24) - 8, 1 << 24, (1 << 24) + 3):
        for a, b in zip(mx.mxfp4_linear_backward(_far(dev, dy, stride), weight), want):
            assert torch.equal(a, b)


def test_far_gradients_take_each_tile():
    lib = _lib()
    assert {lib.mxfp4_backward_plan(m, n, k, TYPE_CODE[BF16])["tile"] for m, n, k in
            ((40, 1032, 20001), (70, 520, 300), (130, 64, 40001))} == {(64, 256), (128, 128), (256, 256)}
