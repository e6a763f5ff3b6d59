"""The 4-bit layer on the GPU against its definition in float64 (oracle/mxfp4_block.py): quantizers bit for bit, products within
bounds derived from the arithmetic.

Bounds. u(t) is half a step of the output type (torch.finfo(t).eps / 2), the last rounding. A block's 32 products are whole
multiples of one power of two below 2^13 of it: their sum is exact. An instruction adds two or four blocks' sums to a
float32 and cuts each below 2^-22 of the largest of them, at most 5 cuts: with S = sum |p|, which bounds every partial sum,
|error| <= ceil(K / 64) * 5 * 2^-22 S (twice that where K is split and joined, whose additions round by 2^-24 each). As a norm
the cuts are held to half of 5 * 2^-22 |y| per 64 columns.

The input's gradient sums exact bfloat16 products in float32: one rounding of 2^-24 per addend at most, of which there are
N times 1, 2 or 3 parts: |error| <= 2^-24 (parts N + 2) S, and, as a norm, 2^-19 |dx| (N / 16 roundings of independent sign).
"""

from __future__ import annotations

import pytest
import torch

from oracle import mxfp4_block as ob

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]
CODES, SCALE = torch.float4_e2m1fn_x2, torch.float8_e8m0fnu


def _mx():
    import mx_qlinear

    return mx_qlinear


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _acts(m, k, dtype, seed, spread=1.0):
    g = _gen(seed)
    x = torch.randn(m, k, generator=g) * torch.exp(spread * torch.randn(m, 1, generator=g))
    return x.to(dtype)


def _half_step(dtype):
    return torch.finfo(dtype).eps / 2


def _same(a, b):
    """Equal values, NaN where NaN."""
    return torch.equal(a.isnan(), b.isnan()) and torch.equal(torch.nan_to_num(a, 0.0, 1e300, -1e300),
                                                             torch.nan_to_num(b, 0.0, 1e300, -1e300))


def check_product(y, xv, wv, bias):
    """y against float64 values xv [M, K] and wv [N, K] of the operands."""
    b = 0 if bias is None else bias.double()
    ref = xv @ wv.t() + b
    got = y.double().cpu()
    assert got.shape == ref.shape
    u, k = _half_step(y.dtype), xv.shape[1]
    cuts = -(-k // 64) * 5 * 2.0**-22
    bound = u * ref.abs() + torch.finfo(y.dtype).tiny + 2 * cuts * (xv.abs() @ wv.abs().t())
    bound += 2.0**-23 * (ref.abs() + (0 if bias is None else b.abs()))  # the bias's addition
    err = (got - ref).abs()
    assert bool((err <= bound * (1 + u)).all()), f"worst {float((err / bound).max())} of the bound"
    if ref.numel() >= 4096 and bool(torch.isfinite(ref).all()):
        assert float(err.norm() / ref.norm()) <= u + cuts / 2 + 2.0**-23


# ---------------------------------------------------------------------------------------
# quantizer
# ---------------------------------------------------------------------------------------

SIZES = [(1, 1), (1, 8), (2, 31), (3, 32), (3, 33), (5, 130), (17, 1000), (33, 640), (64, 4999), (257, 2048), (9, 20480)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,k", SIZES)
def test_rows_codes_and_scales(dev, dtype, m, k):
    mx = _mx()
    x = _acts(m, k, dtype, m * 7919 + k, 3.0)
    q, s = mx.quantize_mxfp4(x.to(dev))
    assert q.dtype == CODES and s.dtype == SCALE and q.shape == (m, -(-k // 2)) and s.shape == (m, -(-k // 32))
    want, b, codes = ob.rows(x)
    assert torch.equal(s.cpu().contiguous().view(torch.uint8).int(), b)
    assert torch.equal(q.cpu().contiguous().view(torch.uint8), ob.pack(codes))
    for out in DTYPES:
        back = mx.dequantize_mxfp4(q, s, out, width=k)
        assert torch.equal(back.cpu(), want.to(out))
    # contiguous copies of the pair give the same
    assert torch.equal(mx.dequantize_mxfp4(q.contiguous(), s.contiguous(), torch.float32, width=k).cpu(), want.float())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_every_16_bit_value(dev, dtype):
    """All 65,536 inputs, each in a block of its own magnitude's neighbours."""
    mx = _mx()
    x = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(dtype).view(512, 128)
    q, s = mx.quantize_mxfp4(x.to(dev))
    want, b, codes = ob.rows(x.double())
    assert torch.equal(s.cpu().view(torch.uint8).int(), b)
    assert torch.equal(q.cpu().view(torch.uint8), ob.pack(codes))
    assert _same(mx.dequantize_mxfp4(q, s, torch.float32).cpu().double(), want.float().double())


@pytest.mark.parametrize("dtype", DTYPES)
def test_edges_of_a_block(dev, dtype):
    """Zeros, the borders of the exponent's choice, ties, the smallest and largest magnitudes, NaN and infinities."""
    mx = _mx()
    top, tiny = torch.finfo(dtype).max, torch.finfo(dtype).smallest_normal
    rows = torch.zeros(16, 96, dtype=torch.float64)
    rows[1, 0] = 6.0
    rows[2, 0] = 6.0 * (1 + 2.0**-7)
    rows[3, :8] = torch.tensor([6.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])  # ties at e = 0
    rows[4, :8] = -rows[3, :8]
    rows[5, 0], rows[5, 1] = top, top / 16
    rows[6, 5] = float("nan")
    rows[7, 35], rows[7, 36] = float("inf"), 3.0
    rows[8, :] = float("-inf")
    rows[9, 64], rows[9, 10] = float("nan"), -7.0
    rows[10, 0], rows[10, 1] = tiny, tiny / 4  # and subnormal
    rows[11, :] = tiny / 8
    rows[12, :] = -0.0
    rows[13, 0], rows[13, 1] = 1.0, 2.0**-20  # far below the block's largest
    rows[14, 0], rows[14, 1] = 4.0 + 2.0**-5, 5.0
    rows[15, 95] = -0.24
    x = rows.to(dtype)
    q, s = mx.quantize_mxfp4(x.to(dev))
    want, b, codes = ob.rows(x)
    assert torch.equal(s.cpu().view(torch.uint8).int(), b)
    assert torch.equal(q.cpu().view(torch.uint8), ob.pack(codes))
    assert _same(mx.dequantize_mxfp4(q, s, torch.float32).cpu().double(), want.float().double())


def test_quantizer_takes_any_layout(dev):
    mx = _mx()
    base = _acts(12, 700, torch.bfloat16, 3)
    on = base.to(dev)
    for view, host in ((on[:, 3:200], base[:, 3:200]), (on[::2, 1:98], base[::2, 1:98]), (on.t()[:50], base.t()[:50]),
                       (on[:1].expand(5, 700), base[:1].expand(5, 700)), (on.view(3, 4, 700)[:, 1], base.view(3, 4, 700)[:, 1]),
                       (on.view(3, 4, 700)[..., :33], base.view(3, 4, 700)[..., :33]), (on[5], base[5])):
        q, s = mx.quantize_mxfp4(view)
        k = host.shape[-1]
        assert q.shape == (*host.shape[:-1], -(-k // 2)) and s.shape == (*host.shape[:-1], -(-k // 32))
        _, b, codes = ob.rows(host.reshape(-1, k))
        assert torch.equal(q.cpu().contiguous().view(torch.uint8).reshape(-1, -(-k // 2)), ob.pack(codes))
        assert torch.equal(s.cpu().contiguous().view(torch.uint8).reshape(-1, -(-k // 32)).int(), b)
        back = mx.dequantize_mxfp4(q, s, torch.float32, width=k)
        assert back.shape == host.shape
    q, s = mx.quantize_mxfp4(on[:0])
    assert q.shape == (0, 350) and mx.dequantize_mxfp4(q, s).shape == (0, 700)


def test_foreign_pairs_are_restored(dev):
    """Every code under every scale byte, from rows that are slices at odd places."""
    mx = _mx()
    q = torch.arange(16, dtype=torch.uint8).repeat(256, 2)
    q = (q | (q.flip(1) << 4)).contiguous()  # [256, 32]: 64 columns
    s = torch.arange(256, dtype=torch.uint8)[:, None].expand(256, 2).contiguous()
    want = ob.values(q, s, 64)
    for out in DTYPES:
        back = mx.dequantize_mxfp4(q.to(dev).view(CODES), s.to(dev).view(SCALE), out)
        assert _same(back.cpu().double(), want.to(out).double())
    wide = torch.zeros(256, 37, dtype=torch.uint8)
    wide[:, 3:35] = q
    ws = torch.zeros(256, 5, dtype=torch.uint8)
    ws[:, 1:3] = s
    back = mx.dequantize_mxfp4(wide.to(dev)[:, 3:35].view(CODES), ws.to(dev)[:, 1:3].view(SCALE), torch.float32, width=63)
    assert _same(back.cpu().double(), want[:, :63].float().double())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,k", [(1, 1), (31, 32), (33, 515), (70, 1000), (130, 4096)])
def test_prepared_weights(dev, dtype, n, k):
    """From floats and from codes: the same bytes where the products read them, zeros behind the columns, 127 or any finite byte
    behind the blocks."""
    mx = _mx()
    w = _acts(n, k, dtype, n + k, 2.0)
    _, b, codes = ob.rows(w)
    a = mx.prepare_mxfp4_weight(w.to(dev))
    q, s = ob.pack(codes), b.to(torch.uint8)
    if k % 2:
        q[:, -1] |= 0xA0  # (what stands behind an odd row is not the weight's)
    c = mx.prepare_mxfp4_weight(q.to(dev).view(CODES), s.to(dev).view(SCALE), in_features=k)
    want = torch.zeros(n, -(-k // 512) * 256, dtype=torch.uint8)
    want[:, : -(-k // 2)] = ob.pack(codes)
    places = ob.tiles(b, k)
    for form in (a, c):
        assert (form.out_features, form.in_features) == (n, k)
        assert torch.equal(form.q.cpu(), want)
        got = form.scale.cpu()
        assert all(int(got[at]) == byte for at, byte in places.items())
        rows = got.view(-1, -(-k // 512), 2, 32, 8).permute(0, 3, 1, 2, 4).reshape(-1, -(-k // 512) * 16)[:n]
        assert bool((rows != 255).all())
    again = mx.prepare_mxfp4_weight(w.to(dev))
    assert torch.equal(a.scale, again.scale) and torch.equal(a.q, again.q)


# ---------------------------------------------------------------------------------------
# products
# ---------------------------------------------------------------------------------------

PRODUCTS = [(1, 1, 1), (1, 16, 32), (1, 100, 5000), (2, 33, 257), (7, 300, 520), (15, 17, 1000), (16, 2049, 640), (17, 64, 33),
            (31, 129, 31), (33, 257, 255), (64, 96, 4096), (100, 520, 1025), (130, 130, 5120), (257, 300, 256), (300, 1000, 777),
            (600, 260, 2048), (1100, 513, 100), (5, 33, 20480), (16, 70, 9000), (16, 40, 20480)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k", PRODUCTS)
def test_linear(dev, dtype, m, n, k):
    mx = _mx()
    x, w = _acts(m, k, dtype, m + k), _acts(n, k, dtype, n + 3 * k, 0.5)
    bias = torch.randn(n, generator=_gen(n)).to(dtype) if (m + n + k) % 2 else None
    xv, wv = ob.rows(x)[0], ob.rows(w)[0]
    weight = mx.prepare_mxfp4_weight(w.to(dev))
    on = None if bias is None else bias.to(dev)
    y = mx.mxfp4_linear(x.to(dev), weight, on)
    assert y.dtype == dtype
    check_product(y, xv, wv, bias)
    z = mx.mxfp4_linear_prequantized(*mx.quantize_mxfp4(x.to(dev)), weight, on, dtype)
    check_product(z, xv, wv, bias)
    if m > 16:
        assert torch.equal(y, z)
    assert torch.equal(mx.mxfp4_linear(x.to(dev), weight, on), y)  # (the same bits on every run)


@pytest.mark.parametrize("out", DTYPES)
@pytest.mark.parametrize("m", [3, 40, 300])
def test_output_types_and_layouts(dev, out, m):
    mx = _mx()
    base, w = _acts(m, 900, torch.bfloat16, 5), _acts(72, 600, torch.bfloat16, 6)
    weight = mx.prepare_mxfp4_weight(w.to(dev))
    x = base.to(dev)[:, 7:607]
    xv, wv = ob.rows(base[:, 7:607])[0], ob.rows(w)[0]
    bias = torch.randn(72, generator=_gen(9))
    check_product(mx.mxfp4_linear(x, weight, bias.to(dev), out), xv, wv, bias.to(out))
    lead = mx.mxfp4_linear(x.unflatten(0, (1, m)), weight, None, out)
    assert lead.shape == (1, m, 72)
    check_product(lead[0], xv, wv, None)
    one = mx.mxfp4_linear(x[0], weight, None, out)
    assert one.shape == (72,)
    check_product(one[None], xv[:1], wv, None)
    assert mx.mxfp4_linear(x[:0], weight, None, out).shape == (0, 72)


@pytest.mark.parametrize("m", [5, 50, 300])
@pytest.mark.parametrize("k", [95, 256, 600, 1024])
def test_foreign_pairs_are_multiplied(dev, m, k):
    """Codes and scales of other making: slices at odd places, any scale bytes within float32's range, a stray last code."""
    mx = _mx()
    g = _gen(m * k)
    half, kb, n = -(-k // 2), -(-k // 32), 70
    q = torch.randint(0, 256, (m, half + 9), generator=g).to(torch.uint8)
    s = torch.randint(110, 140, (m, kb + 3), generator=g).to(torch.uint8)
    wq = torch.randint(0, 256, (n, half), generator=g).to(torch.uint8)
    ws = torch.randint(110, 140, (n, kb), generator=g).to(torch.uint8)
    xv, wv = ob.values(q[:, 5:5 + half], s[:, 1:1 + kb], k), ob.values(wq, ws, k)
    weight = mx.prepare_mxfp4_weight(wq.to(dev).view(CODES), ws.to(dev).view(SCALE), in_features=k)
    y = mx.mxfp4_linear_prequantized(q.to(dev)[:, 5:5 + half].view(CODES), s.to(dev)[:, 1:1 + kb].view(SCALE), weight, None, torch.float32)
    check_product(y, xv, wv, None)
    whole = mx.mxfp4_linear_prequantized(q.to(dev)[:, :half].contiguous().view(CODES), s.to(dev)[:, :kb].contiguous().view(SCALE), weight,
                                         None, torch.float32)
    check_product(whole, ob.values(q[:, :half], s[:, :kb], k), wv, None)


def test_all_scale_bytes_multiply(dev):
    """Row i has the scale byte i in all of its blocks, the weight's rows 127 (and what brings the product back)."""
    mx = _mx()
    g = _gen(4)
    q = torch.randint(0, 256, (255, 64), generator=g).to(torch.uint8)
    wq = torch.randint(0, 256, (32, 64), generator=g).to(torch.uint8)
    s = torch.arange(255, dtype=torch.uint8)[:, None].expand(255, 4).contiguous()
    for byte in (127, 20, 230):
        ws = torch.full((32, 4), byte, dtype=torch.uint8)
        weight = mx.prepare_mxfp4_weight(wq.to(dev).view(CODES), ws.to(dev).view(SCALE))
        y = mx.mxfp4_linear_prequantized(q.to(dev).view(CODES), s.to(dev).view(SCALE), weight, None, torch.float32).cpu().double()
        ref = ob.values(q, s, 128) @ ob.values(wq, ws, 128).t()
        # (partial sums are bounded by the sum of magnitudes, not by the result: below 2^126 of it none overflows, above 2^-100
        # a subnormal one is below 2^-26 of it)
        size = ob.values(q, s, 128).abs() @ ob.values(wq, ws, 128).abs().t()
        fine = (size < 2.0**126) & (size > 2.0**-100)
        assert bool(((y - ref).abs() <= 2 * 5 * 2.0**-22 * size)[fine].all())
        over = ref.abs() > 2.0**129
        assert bool((~torch.isfinite(y))[over].all())


def test_blocks_of_far_magnitudes(dev):
    """Neighbouring blocks up to 2^40 apart: cut as stated, nothing worse; equal and opposite blocks cancel."""
    mx = _mx()
    g = _gen(8)
    x = torch.randn(40, 640, generator=g) * torch.exp2(torch.randint(-20, 21, (40, 20), generator=g).float()).repeat_interleave(32, 1)
    w = torch.randn(50, 640, generator=g)
    xv, wv = ob.rows(x)[0], ob.rows(w)[0]
    weight = mx.prepare_mxfp4_weight(w.to(dev))
    for rows in (slice(0, 40), slice(0, 9)):
        y = mx.mxfp4_linear(x[rows].to(dev), weight).cpu().double()
        ref = xv[rows] @ wv.t()
        bound = 11 * 5 * 2.0**-21 * (xv[rows].abs() @ wv.abs().t()) + 2.0**-24 * ref.abs()
        assert bool(((y - ref).abs() <= bound).all())
    x2 = torch.cat((x[:, :320], x[:, :320]), 1)
    w2 = torch.cat((w[:, :320], -w[:, :320]), 1)
    y = mx.mxfp4_linear(x2.to(dev), mx.prepare_mxfp4_weight(w2.to(dev))).cpu().double()
    bound = 11 * 5 * 2.0**-21 * (ob.rows(x2)[0].abs() @ ob.rows(w2)[0].abs().t())
    assert bool((y.abs() <= bound).all())


@pytest.mark.parametrize("m", [2, 16, 40, 300])
def test_nan_and_infinities_stay_in_their_rows(dev, m):
    mx = _mx()
    x, w = _acts(m, 700, torch.bfloat16, 2), _acts(90, 700, torch.bfloat16, 3)
    clean = mx.mxfp4_linear(x.to(dev), mx.prepare_mxfp4_weight(w.to(dev))).cpu()
    x[1, 699], w[5, 100], w[64, 0] = float("nan"), float("inf"), float("-inf")
    y = mx.mxfp4_linear(x.to(dev), mx.prepare_mxfp4_weight(w.to(dev))).cpu()
    bad = torch.zeros(m, 90, dtype=torch.bool)
    bad[1], bad[:, 5], bad[:, 64] = True, True, True
    assert bool(y[bad].isnan().all()) and torch.equal(y[~bad], clean[~bad])


# ---------------------------------------------------------------------------------------
# the input's gradient
# ---------------------------------------------------------------------------------------

BACKWARD = [(40, 2100, 1300), (64, 5000, 260), (33, 130, 4097), (1, 1, 1), (1, 520, 300), (3, 7, 33), (16, 64, 1000), (33, 130, 100), (70, 257, 511), (300, 96, 1000), (257, 1000, 256),
            (600, 513, 130), (130, 2050, 257), (1100, 72, 40)]
PARTS = {torch.bfloat16: 1, torch.float16: 2, torch.float32: 3}


def check_gradients(dx, db, dy, wv):
    u, n = _half_step(dx.dtype), wv.shape[0]
    dyd = dy.double()
    ref = dyd @ wv
    got = dx.double().cpu()
    assert got.shape == ref.shape
    bound = u * ref.abs() + torch.finfo(dx.dtype).tiny + 2.0**-24 * (PARTS[dx.dtype] * n + 2) * (dyd.abs() @ wv.abs())
    err = (got - ref).abs()
    assert bool((err <= bound * (1 + u)).all()), f"worst {float((err / bound).max())} of the bound"
    if ref.numel() >= 4096:
        assert float(err.norm() / ref.norm()) <= u + 2.0**-19
    if db is not None:
        ref = dyd.sum(0)
        bound = _half_step(db.dtype) * ref.abs() + 2.0**-24 * (dy.shape[0] + 2) * dyd.abs().sum(0)
        assert bool(((db.double().cpu() - ref).abs() <= bound * (1 + u)).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k", BACKWARD)
def test_linear_backward(dev, dtype, m, n, k):
    mx = _mx()
    dy, w = _acts(m, n, dtype, m + n) * 1e-2, _acts(n, k, dtype, n + k, 0.5)
    wv = ob.rows(w)[0]
    weight = mx.prepare_mxfp4_weight(w.to(dev))
    dx, db = mx.mxfp4_linear_backward(dy.to(dev), weight)
    assert dx.dtype == dtype and db.dtype == torch.float32
    check_gradients(dx, db, dy, wv)
    again, none = mx.mxfp4_linear_backward(dy.to(dev), weight, (True, False))
    assert none is None and torch.equal(again, dx)
    none, again = mx.mxfp4_linear_backward(dy.to(dev), weight, (False, True), dtype)
    assert none is None and again.dtype == dtype
    assert mx.mxfp4_linear_backward(dy.to(dev), weight, (False, False)) == (None, None)


@pytest.mark.parametrize("dtype", DTYPES)
def test_gradient_layouts(dev, dtype):
    """Slices at odd places, strided rows, leading dimensions, one row, no rows."""
    mx = _mx()
    base, w = _acts(44, 300, dtype, 1), _acts(104, 333, dtype, 2)
    wv, weight = ob.rows(w)[0], mx.prepare_mxfp4_weight(w.to(dev))
    on = base.to(dev)
    for view, host in ((on[:, 5:109], base[:, 5:109]), (on[::2, 8:112], base[::2, 8:112]), (on.t()[:104].t(), base.t()[:104].t()),
                       (on[:1, 196:], base[:1, 196:]), (on[:1, :104].expand(9, 104), base[:1, :104].expand(9, 104))):
        check_gradients(*mx.mxfp4_linear_backward(view, weight), host, wv)
    dx, db = mx.mxfp4_linear_backward(on[:, :104].unflatten(0, (4, 11)), weight)
    assert dx.shape == (4, 11, 333)
    check_gradients(dx.flatten(0, 1), db, base[:, :104], wv)
    dx, db = mx.mxfp4_linear_backward(on[0, :104], weight)
    assert dx.shape == (333,)
    dx, db = mx.mxfp4_linear_backward(on[:0, :104], weight)
    assert dx.shape == (0, 333) and bool((db == 0).all())


@pytest.mark.parametrize("dtype", DTYPES)
def test_nan_and_infinities_in_the_gradient(dev, dtype):
    """A row of dx has what its row of dy and the weight's columns bring, no more: neighbours are clean, also behind column N."""
    mx = _mx()
    for n in (100, 104):
        dy, w = _acts(70, n, dtype, 1), _acts(n, 300, dtype, 2)
        clean = mx.mxfp4_linear_backward(dy.to(dev), mx.prepare_mxfp4_weight(w.to(dev)))[0].cpu()
        dy[4, 0], dy[9, n - 1] = float("inf"), float("nan")
        w[n - 1, 40] = float("nan")  # columns 32 .. 63 of that row
        dx = mx.mxfp4_linear_backward(dy.to(dev), mx.prepare_mxfp4_weight(w.to(dev)))[0].cpu()
        fine = torch.ones(70, 300, dtype=torch.bool)
        fine[4], fine[9], fine[:, 32:64] = False, False, False
        assert torch.equal(dx[fine], clean[fine])
        assert bool((~torch.isfinite(dx[4])).all()) and bool(dx[9].isnan().all()) and bool(dx[:, 32:64].isnan().all())


def test_weights_of_all_scale_bytes_pass_gradients(dev):
    """Bytes 2 to 252: below, a value can be subnormal, above, past float32's range (6 * 2^126), whose product with the other
    rows' zeros is NaN."""
    mx = _mx()
    g = _gen(12)
    wq = torch.randint(0, 256, (64, 128), generator=g).to(torch.uint8)
    ws = torch.randint(2, 253, (64, 8), generator=g).to(torch.uint8)
    weight = mx.prepare_mxfp4_weight(wq.to(dev).view(CODES), ws.to(dev).view(SCALE))
    wv = ob.values(wq, ws, 256)
    dy = torch.zeros(64, 64)  # row i picks weight row i
    dy[torch.arange(64), torch.arange(64)] = 1.0
    for dtype in DTYPES[::2]:
        dx = mx.mxfp4_linear_backward(dy.to(dtype).to(dev), weight, (True, False))[0].cpu()
        assert _same(dx.double(), wv.to(dtype).double())


def test_range_of_float32_gradients(dev):
    """Through a weight of ones every value of 24 bits comes back from 2^-103 to bfloat16's largest and half a step; from there on it
    is an infinity."""
    mx = _mx()
    weight = mx.prepare_mxfp4_weight(torch.ones(1, 32, device=dev))
    g = _gen(3)
    mant = 1 + torch.randint(0, 1 << 23, (231, 8), generator=g).double() * 2.0**-23
    mant[:, 0], mant[:, 1] = 2 - 2.0**-23, 1 + 2.0**-23
    dy = mant * torch.exp2(torch.arange(-103, 128).double())[:, None] * torch.tensor([1, 1, 1, 1, -1, -1, -1, 1.0], dtype=torch.float64)
    edge = (2 - 2.0**-8) * 2.0**127
    dy[-1, 2], dy[-1, 3] = edge, edge - 2.0**104
    dy = dy.float().reshape(-1, 1)
    dx = mx.mxfp4_linear_backward(dy.to(dev), weight, (True, False))[0].cpu()
    want = torch.where(dy.double().abs() >= edge, torch.copysign(torch.full_like(dy, float("inf")), dy), dy)
    assert torch.equal(dx, want.expand(-1, 32)) and bool(torch.isinf(want).any())


@pytest.mark.parametrize("m,k", [(1, 4992), (300, 4992), (1100, 4992)])
def test_weights_past_float32_pass_gradients(dev, m, k):
    """Every code under the bytes 250 to 254 (and 2), a layer of one output: below 2^128 the value itself, from there on, which
    begins with code 4 under byte 253, an infinity; in fp16 and fp32 gradients, whose other parts are zeros, NaN as well."""
    mx = _mx()
    wq = torch.arange(256, dtype=torch.uint8).repeat(k // 512 + 1)[None, :k // 2].contiguous()
    ws = torch.tensor([2, 250, 251, 252, 253, 254], dtype=torch.uint8).repeat_interleave(8).repeat(k // 32)[None, :k // 32].contiguous()
    wv = ob.values(wq, ws, k)
    over = wv.abs() >= 2.0**128
    assert bool(((ws == 253).repeat_interleave(32, 1) & over).any()) and not bool(((ws < 253).repeat_interleave(32, 1) & over).any())
    weight = mx.prepare_mxfp4_weight(wq.to(dev).view(CODES), ws.to(dev).view(SCALE))
    for dtype in DTYPES:
        dx = mx.mxfp4_linear_backward(torch.ones(m, 1, dtype=dtype, device=dev), weight, (True, False))[0].double().cpu()
        want = wv.float().to(dtype).double().expand(m, k)
        on = over.expand(m, k)
        assert torch.equal(dx[~on], want[~on])
        if dtype == torch.bfloat16:
            assert torch.equal(dx[on], want[on])
        else:
            assert not bool(torch.isfinite(dx[on]).any())


# ---------------------------------------------------------------------------------------
# graphs, streams, the module
# ---------------------------------------------------------------------------------------

@pytest.mark.parametrize("m", [1, 40, 300])
def test_captured_and_replayed(dev, m):
    mx = _mx()
    x, dy = _acts(m, 600, torch.float16, 1).to(dev), _acts(m, 90, torch.float16, 2).to(dev)
    weight = mx.prepare_mxfp4_weight(_acts(90, 600, torch.float16, 3).to(dev))
    bias = torch.randn(90, generator=_gen(2)).half().to(dev)

    def step():
        pair = mx.quantize_mxfp4(x)
        return (mx.mxfp4_linear(x, weight, bias), mx.mxfp4_linear_prequantized(*pair, weight, bias, torch.float16),
                mx.dequantize_mxfp4(*pair), *mx.mxfp4_linear_backward(dy, weight))

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for seed in range(3):
        x.copy_(_acts(m, 600, torch.float16, 10 + seed))
        dy.copy_(_acts(m, 90, torch.float16, 20 + seed))
        want = step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_module_with_a_float64_bias(dev):
    """As a model cast to float64 has it: taken, and its gradient is float32's."""
    mx = _mx()
    w, x, dy = _acts(70, 300, torch.float32, 1), _acts(9, 300, torch.float32, 2), _acts(9, 70, torch.float32, 3)
    grads = []
    for dtype in (torch.float32, torch.float64):
        layer = mx.Mxfp4Linear.from_weight(w.to(dev), torch.ones(70, device=dev)).to(dtype)
        xx = x.to(dev).requires_grad_()
        layer(xx).backward(dy.to(dev))
        assert layer.bias.grad.dtype == dtype
        grads.append((xx.grad, layer.bias.grad.double()))
    assert torch.equal(grads[0][0], grads[1][0]) and torch.equal(grads[0][1], grads[1][1])


@pytest.mark.parametrize("m", [3, 40])
def test_deterministic_mode(dev, m):
    """Every function and both modules under torch.use_deterministic_algorithms: the same bits."""
    mx = _mx()
    x, r, w = _acts(m, 300, torch.bfloat16, 1).to(dev), _acts(m, 300, torch.bfloat16, 2).to(dev), _acts(70, 300, torch.bfloat16, 3).to(dev)

    def run():
        weight = mx.prepare_mxfp4_weight(w)
        q, s = mx.quantize_mxfp4(x)
        nq, ns, total, rstd = mx.rms_norm_quantize_mxfp4(x, None, 1e-6, residual=r, return_rstd=True)
        n8, s8 = mx.rms_norm_quantize_fp8(x)
        y = mx.mxfp4_linear(x, weight)
        norm, layer = mx.RMSNorm(300, keep_fp8=True, device=dev, dtype=torch.bfloat16), mx.Mxfp4Linear.from_weight(w)
        xx = x.clone().requires_grad_()
        layer(norm(xx)).backward(y)
        return [t.view(torch.uint8) if t.dtype in (CODES, SCALE, torch.float8_e4m3fn) else t for t in
                (weight.q, weight.scale, q, s, nq, ns, total, rstd, n8, s8, y, mx.dequantize_mxfp4(q, s),
                 mx.mxfp4_linear_prequantized(q, s, weight), *mx.mxfp4_linear_backward(y, weight),
                 *mx.rms_norm_backward(x, total, rstd, None, r), xx.grad, norm.weight.grad)]

    want = run()
    torch.use_deterministic_algorithms(True)
    try:
        got = run()
    finally:
        torch.use_deterministic_algorithms(False)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_two_streams_at_once(dev):
    """Calls of different inputs on two streams share no memory."""
    mx = _mx()
    weight = mx.prepare_mxfp4_weight(_acts(300, 1000, torch.bfloat16, 3).to(dev))
    xs = [_acts(m, 1000, torch.bfloat16, m).to(dev) for m in (8, 200, 520)]
    want = [mx.mxfp4_linear(x, weight) for x in xs]
    back = [mx.mxfp4_linear_backward(y, weight) for y in want]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for i in range(6):
        with torch.cuda.stream(streams[i % 2]):
            y = mx.mxfp4_linear(xs[i % 3], weight)
            got.append((i % 3, y, mx.mxfp4_linear_backward(y, weight)))
    torch.cuda.synchronize()
    for j, y, (dx, db) in got:
        assert torch.equal(y, want[j]) and torch.equal(dx, back[j][0]) and torch.equal(db, back[j][1])


@pytest.mark.parametrize("dtype", DTYPES)
def test_module_with_an_adapter(dev, dtype):
    """A frozen layer with a trained low-rank adapter and bias: gradients against float64 autograd of the values."""
    mx = _mx()
    m, k, n, r = 50, 320, 96, 8
    w = _acts(n, k, torch.float32, 1, 0.3)
    x0, dy = _acts(m, k, dtype, 2), _acts(m, n, dtype, 3)
    layer = mx.Mxfp4Linear.from_weight(w.to(dev), torch.randn(n, generator=_gen(5)).to(dtype).to(dev))
    assert layer.bias.requires_grad and not layer.qweight.requires_grad
    a = _acts(r, k, dtype, 6, 0.0).to(dev).requires_grad_()
    b = _acts(n, r, dtype, 7, 0.0).to(dev).requires_grad_()
    x = x0.to(dev).requires_grad_()
    y = layer(x) + (x @ a.t()) @ b.t()
    y.backward(dy.to(dev))
    xv, wv = ob.rows(x0)[0], ob.rows(w)[0]
    with torch.no_grad():
        check_product(layer(x), xv, wv, layer.bias.detach().cpu())
    dx, db = mx.mxfp4_linear_backward(dy.to(dev), layer.prepared())
    check_gradients(dx, None, dy, wv)
    ref = dy.double() @ wv + dy.double() @ b.detach().cpu().double() @ a.detach().cpu().double()
    # the adapter's own path rounds (dy b) and its product to the type, and their sum once more: 4 steps of its magnitude
    side = (dy.double().abs() @ b.detach().cpu().double().abs()) @ a.detach().cpu().double().abs()
    bound = 4 * _half_step(dtype) * (side + ref.abs() + dyd_abs(dy, wv))
    assert bool(((x.grad.double().cpu() - ref).abs() <= bound).all())
    check_bias = dy.double().sum(0)
    assert bool(((layer.bias.grad.double().cpu() - check_bias).abs() <= 2 * _half_step(dtype) * dy.double().abs().sum(0)).all())


def dyd_abs(dy, wv):
    return 2.0**-8 * (dy.double().abs() @ wv.abs())


def test_module_state_moves(dev):
    mx = _mx()
    layer = mx.Mxfp4Linear.from_weight(_acts(70, 300, torch.bfloat16, 1).to(dev))
    x = _acts(9, 300, torch.bfloat16, 2).to(dev)
    want = layer(x)
    other = mx.Mxfp4Linear(300, 70, bias=False, device=dev)
    assert bool((other(x) == 0).all())
    other.load_state_dict(layer.state_dict())
    assert torch.equal(other(x), want)
    assert torch.equal(other.cpu().to(dev)(x), want)
    import copy

    assert torch.equal(copy.deepcopy(layer)(x), want)


def test_gradient_against_differences(dev):
    """dx of the layer taken as the linear map of the held weight: differences of float32 outputs of inputs that 4 bits hold."""
    mx = _mx()
    g = _gen(3)
    w = _acts(24, 64, torch.float32, 4)
    weight = mx.prepare_mxfp4_weight(w.to(dev))
    x = torch.zeros(2, 64)
    x[:, 0], x[:, 32] = 6.0, 6.0  # (the blocks' scale is 1 whatever the others are)
    dy = torch.randn(2, 24, generator=g)
    dx = mx.mxfp4_linear_backward(dy.to(dev), weight, (True, False))[0].cpu()
    for j in (1, 5, 31, 33, 63):
        up, down = x.clone(), x.clone()
        up[:, j], down[:, j] = 2.0, -2.0
        d = (mx.mxfp4_linear(up.to(dev), weight) - mx.mxfp4_linear(down.to(dev), weight)).cpu().double() / 4.0
        want = (d * dy.double()).sum(1)
        size = (dy.double().abs() * 12 * ob.rows(w)[0].abs().sum(1)).sum(1)
        assert bool(((dx[:, j].double() - want).abs() <= 2.0**-20 * size).all())


def test_modules_are_not_captured(dev):
    mx = _mx()
    layer = mx.Mxfp4Linear.from_weight(_acts(64, 256, torch.bfloat16, 1).to(dev), torch.zeros(64, dtype=torch.bfloat16, device=dev))
    x = _acts(32, 256, torch.bfloat16, 2).to(dev)
    with torch.no_grad():
        want = layer(x)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="not captured"):
            layer(x)
        with torch.no_grad():
            y = layer(x)
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want)


def test_pairs_in_any_order(dev):
    """Transposed and strided codes and scales, and leading dimensions that no view merges."""
    mx = _mx()
    g = _gen(8)
    q = torch.randint(0, 256, (40, 5, 32), generator=g).to(torch.uint8)
    s = torch.randint(120, 131, (40, 5, 2), generator=g).to(torch.uint8)
    wq = torch.randint(0, 256, (48, 32), generator=g).to(torch.uint8)
    ws = torch.randint(120, 131, (48, 2), generator=g).to(torch.uint8)
    wv = ob.values(wq, ws, 64)
    turned = (wq.t().contiguous().to(dev).t().view(CODES), ws.t().contiguous().to(dev).t().view(SCALE))
    weight = mx.prepare_mxfp4_weight(*turned)
    plain = mx.prepare_mxfp4_weight(wq.to(dev).view(CODES), ws.to(dev).view(SCALE))
    assert torch.equal(weight.q, plain.q)
    assert torch.equal(mx.dequantize_mxfp4(*turned, torch.float32).cpu().double(), wv)
    for order in ((0, 1, 2), (1, 0, 2)):
        qv, sv = q.permute(order), s.permute(order)
        xv = ob.values(qv.reshape(200, 32), sv.reshape(200, 2), 64)
        pair = (q.to(dev).permute(order).view(CODES), s.to(dev).permute(order).view(SCALE))
        assert torch.equal(mx.dequantize_mxfp4(*pair, torch.float32).cpu().double(), xv.view(*qv.shape[:2], 64))
        y = mx.mxfp4_linear_prequantized(*pair, weight, None, torch.float32)
        assert y.shape == (*qv.shape[:2], 48)
        check_product(y.reshape(200, 48), xv, wv, None)


def test_a_layer_made_in_inference_mode_trains(dev):
    mx = _mx()
    w, x0 = _acts(40, 96, torch.bfloat16, 1), _acts(20, 96, torch.bfloat16, 2)
    with torch.inference_mode():
        layer = mx.Mxfp4Linear.from_weight(w.to(dev), torch.zeros(40, dtype=torch.bfloat16, device=dev))
    x = x0.to(dev).requires_grad_()
    y = layer(x)
    dy = torch.ones_like(y)
    y.backward(dy)
    check_gradients(x.grad, layer.bias.grad, dy.cpu(), ob.rows(w)[0])


def test_more_than_2_to_the_32_elements(dev):
    """Rows on both sides of every power of two that an offset could be cut at, against the same rows by themselves."""
    mx = _mx()
    m, k = 135_000, 32_768  # 4.4e9 elements
    x = torch.empty(m, k, dtype=torch.bfloat16, device=dev)
    for i in range(0, m, 27_000):
        x[i:i + 27_000].normal_()
    at = sorted({0, m - 1, *(min(m - 1, 2**p // w + d) for p in (29, 30, 31, 32) for w in (k // 2, k, 2 * k) for d in (-1, 0, 1))})
    at = torch.tensor([i for i in at if 0 <= i < m])
    few = x[at.to(dev)]
    q, s = mx.quantize_mxfp4(x)
    del x
    _, b, codes = ob.rows(few.cpu())
    assert torch.equal(q.view(torch.uint8)[at.to(dev)].cpu(), ob.pack(codes))
    assert torch.equal(s.view(torch.uint8)[at.to(dev)].cpu().int(), b)
    back = mx.dequantize_mxfp4(q, s)
    assert torch.equal(back[at.to(dev)].cpu().double(), ob.rows(few.cpu())[0])
    del back
    w = _acts(40, k, torch.bfloat16, 4)
    y = mx.mxfp4_linear_prequantized(q, s, mx.prepare_mxfp4_weight(w.to(dev)))
    check_product(y[at.to(dev)], ob.rows(few.cpu())[0], ob.rows(w)[0], None)


def test_products_of_more_than_2_to_the_32_elements(dev):
    mx = _mx()
    m, n, k = 135_000, 32_768, 64
    w = _acts(n, k, torch.bfloat16, 4, 0.5)
    weight = mx.prepare_mxfp4_weight(w.to(dev))
    x = torch.randn(m, k, device=dev, dtype=torch.bfloat16)
    at = sorted({0, m - 1, *(min(m - 1, 2**p // n + d) for p in (29, 30, 31, 32) for d in (-1, 0, 1))})
    at = torch.tensor([i for i in at if 0 <= i < m])
    wv = ob.rows(w)[0]
    y = mx.mxfp4_linear(x, weight)
    check_product(y[at.to(dev)], ob.rows(x[at.to(dev)].cpu())[0], wv, None)
    dx, db = mx.mxfp4_linear_backward(y, weight)  # (y as the gradient: 4.4e9 elements)
    check_gradients(dx[at.to(dev)], None, y[at.to(dev)].cpu(), wv)
    total, size = torch.zeros(n, dtype=torch.float64, device=dev), torch.zeros(n, dtype=torch.float64, device=dev)
    for i in range(0, m, 13_500):
        part = y[i:i + 13_500].double()
        total += part.sum(0)
        size += part.abs().sum(0)
    assert bool(((db.double() - total).abs() <= 2.0**-24 * (m + 2) * size).all())
    del dx, db, x
    turned = mx.prepare_mxfp4_weight(_acts(k, n, torch.bfloat16, 5, 0.5).to(dev))  # (and a gradient of as many)
    dy = torch.randn(m, k, device=dev, dtype=torch.float16)
    dx, _ = mx.mxfp4_linear_backward(dy, turned)
    check_gradients(dx[at.to(dev)], None, dy[at.to(dev)].cpu(), ob.rows(_acts(k, n, torch.bfloat16, 5, 0.5))[0])


def test_module_gives_the_gradients_asked_for(dev):
    """Only the bias's, only the input's, none of either, and those of no rows."""
    mx = _mx()
    w, bias = _acts(40, 96, torch.bfloat16, 1), _acts(1, 40, torch.bfloat16, 2)[0]
    layer = mx.Mxfp4Linear.from_weight(w.to(dev), bias.to(dev))
    x0, dy = _acts(20, 96, torch.bfloat16, 3), _acts(20, 40, torch.bfloat16, 4)
    want_x, want_b = mx.mxfp4_linear_backward(dy.to(dev), layer.prepared(), grad_dtype=torch.bfloat16)
    for of_x in (False, True):
        for of_b in (False, True):
            x = x0.to(dev).requires_grad_(of_x)
            layer.bias.requires_grad_(of_b).grad = None
            y = layer(x)
            assert y.requires_grad == (of_x or of_b)
            if y.requires_grad:
                y.backward(dy.to(dev))
            assert (x.grad is None) == (not of_x) and (not of_x or torch.equal(x.grad, want_x))
            assert (layer.bias.grad is None) == (not of_b) and (not of_b or torch.equal(layer.bias.grad, want_b))
    x = x0[:0].to(dev).requires_grad_()
    layer.bias.grad = None
    layer(x).sum().backward()
    assert x.grad.shape == (0, 96) and bool((layer.bias.grad == 0).all())
    with torch.no_grad():
        x = x0.to(dev).requires_grad_()
        assert not layer(x).requires_grad
