"""8-bit floating point layer on the GPU against its definition in float64 (oracle/fp8_block.py): quantizers bit for bit,
products within bounds derived from the arithmetic.

Bounds. u(t) is half a step of the output type (bf16 2^-8 / 2 ..., i.e. torch.finfo(t).eps / 2), the last rounding. In
front of it, float32 outputs (and all of up to 16 rows) sum exact bf16 x bf16 products in float32: at most one rounding
of 2^-24 per addend, so |error| <= 2^-24 (K + 2) sum|p|. bf16 and fp16 outputs of more rows go through the e4m3
instruction, which cuts each addend of a 64-long sum below 2^-13 of the largest: |error| <= 64 * 2^-13 max|p| per 64.
Those are worst cases; the norms are held to (u + 2^-10) |y|, with cuts of independent sign (rms of a cut 2^-13 max|p|,
max|p| <= 8 rms(p) over 64 products of normal values), and float32 to 2^-19 |y| (K / 16 roundings of independent sign).
"""

from __future__ import annotations

import pytest
import torch

from oracle import fp8_block as ob

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


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


def _chunk_max(v, n=64):
    m, k = v.shape
    p = torch.zeros(m, -(-k // n) * n, dtype=torch.float64)
    p[:, :k] = v.abs()
    return p.view(m, -1, n).amax(-1)


def check_product(y, xv, wv, bias, wide):
    """y against float64 values xv [M, K] and wv [N, K] of the operands."""
    ref = xv @ wv.t() + (0 if bias is None else bias.double())
    got = y.double().cpu()
    assert got.shape == ref.shape
    u, k = _half_step(y.dtype), xv.shape[1]
    bound = u * ref.abs() + torch.finfo(y.dtype).tiny
    bound += 2.0**-24 * (k + 2) * (xv.abs() @ wv.abs().t() + (0 if bias is None else bias.double().abs()))
    if not wide:
        bound += 64 * 2.0**-13 * (_chunk_max(xv) @ _chunk_max(wv).t())
    err = (got - ref).abs()
    assert bool((err <= bound * (1 + u)).all()), f"worst {float((err / bound).max())} of the bound"
    if ref.numel() >= 4096 and bool(torch.isfinite(ref).all()):
        tol = 2.0**-19 + u if y.dtype == torch.float32 or wide else u + 2.0**-10
        assert float(err.norm() / ref.norm()) <= tol


# ---------------------------------------------------------------------------------------
# quantizers
# ---------------------------------------------------------------------------------------

SIZES = [(1, 1), (1, 8), (2, 127), (3, 128), (3, 129), (5, 130), (17, 1000), (33, 640), (64, 4999), (257, 2048), (9, 20480)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,k", SIZES)
def test_rows_codes_and_scales(dev, dtype, m, k):
    mx = _mx()
    x = _acts(m, k, dtype, m * 7919 + k, 3.0)
    q, s = mx.quantize_fp8_block128(x.to(dev))
    assert q.shape == x.shape and s.shape == (m, -(-k // 128))
    want, e = ob.rows(x)
    assert torch.equal(s.cpu().contiguous().view(torch.uint8).int() - 127, e)
    assert torch.equal(ob.values(q, s), want)
    for out in DTYPES:
        back = mx.dequantize_fp8_block128(q, s, out)
        assert torch.equal(back.cpu(), want.to(out))
    # contiguous copies of the pair give the same
    assert torch.equal(mx.dequantize_fp8_block128(q.contiguous(), s.contiguous(), torch.float32).cpu(), want.float())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_every_16_bit_value(dev, dtype):
    """All 65,536 inputs, each in a block of its own magnitude's neighbours."""
    mx = _mx()
    x = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(dtype).view(512, 128)
    q, s = mx.quantize_fp8_block128(x.to(dev))
    want, e = ob.rows(x.double())
    assert torch.equal(s.cpu().view(torch.uint8).int() - 127, e)
    assert _same(ob.values(q, s), want)


@pytest.mark.parametrize("dtype", DTYPES)
def test_edges_of_a_block(dev, dtype):
    """Zeros, the borders of the exponent's choice, ties, the smallest and largest magnitudes, NaN and infinities."""
    mx = _mx()
    top = torch.finfo(dtype).max
    rows = torch.zeros(14, 256, dtype=torch.float64)
    rows[1, 0] = 448.0
    rows[2, 0] = 448.5 if dtype != torch.bfloat16 else 450.0
    rows[3, :4] = torch.tensor([448.0, 1.0625, 1.1875, -1.0625])  # ties at e = 0
    rows[4, 0] = torch.finfo(dtype).tiny
    rows[5, 0], rows[5, 1] = top, top / 1024
    rows[6, 5] = float("nan")
    rows[7, 5], rows[7, 6] = float("inf"), 3.0
    rows[8, :] = float("-inf")
    rows[9, 130], rows[9, 131] = float("nan"), -7.0
    rows[10, 0] = torch.finfo(dtype).smallest_normal / 4  # subnormal
    rows[11, :] = -1.75
    rows[12, :] = -0.0
    rows[13, 0], rows[13, 1] = 1.0, 2.0**-20  # far below the block's largest
    x = rows.to(dtype)
    q, s = mx.quantize_fp8_block128(x.to(dev))
    want, e = ob.rows(x)
    assert torch.equal(s.cpu().view(torch.uint8).int() - 127, e)
    assert _same(ob.values(q, s), want)
    back = mx.dequantize_fp8_block128(q, s, torch.float32).cpu()
    assert _same(back.double(), want.float().double())
    assert bool((s.cpu().view(torch.uint8) < 255).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,k", [(1, 1), (128, 128), (130, 205), (300, 130), (1000, 217), (513, 1152)])
def test_weight_tiles(dev, dtype, n, k):
    mx = _mx()
    w = (_acts(n, k, torch.float32, n + k, 2.0) * 0.02).to(dtype)
    if n > 2:
        w[1, 0], w[n - 1, k - 1] = float("nan"), float("inf")
    want, e = ob.tiles(w)
    p = mx.prepare_fp8_weight(w.to(dev))
    nb, kb = e.shape
    assert torch.equal(p.scale[:, :kb].cpu().view(torch.uint8).int() - 127, e)
    assert torch.equal(p.scale_t[:, :nb].cpu().view(torch.uint8).int() - 127, e.t())
    assert _same(ob.values(p.q, p.scale[:, :kb], 128)[:, :k], want)
    assert _same(ob.values(p.qt, p.scale_t[:, :nb], 128)[:, :n], want.t())
    # behind the weight's columns the products read zeros
    assert bool((p.q[:, k:].cpu().view(torch.uint8) == 0).all()) and bool((p.qt[:, n:].cpu().view(torch.uint8) == 0).all())
    # the stored form gives the same layout
    r = mx.prepare_fp8_weight(p.q[:, :k], p.scale[:, :kb])
    for a, b in ((p.q, r.q), (p.qt, r.qt)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    assert torch.equal(p.scale[:, :kb].view(torch.uint8), r.scale[:, :kb].view(torch.uint8))
    assert torch.equal(p.scale_t[:, :nb].view(torch.uint8), r.scale_t[:, :nb].view(torch.uint8))
    assert mx.prepare_fp8_weight(w.to(dev), transposed=False).qt is None


def test_strided_and_many_dimensional_inputs(dev):
    mx = _mx()
    big = _acts(40, 900, torch.bfloat16, 5).to(dev)
    for view in (big[:, 3:700], big[::2, :256], big[3:], big.t(), big.view(4, 10, 900), big.view(4, 10, 900).transpose(0, 1)):
        q, s = mx.quantize_fp8_block128(view)
        assert q.shape == view.shape
        flat = view.reshape(-1, view.shape[-1]).cpu()
        want, _ = ob.rows(flat)
        assert torch.equal(mx.dequantize_fp8_block128(q, s, torch.float32).cpu().reshape(flat.shape), want.float())
    one = big[0]
    q, s = mx.quantize_fp8_block128(one)
    assert q.shape == (900,) and s.shape == (8,)
    assert torch.equal(mx.dequantize_fp8_block128(q, s).cpu(), ob.rows(one.cpu()[None])[0][0].bfloat16())


# ---------------------------------------------------------------------------------------
# products
# ---------------------------------------------------------------------------------------

# (rows of every path: fused, streamed, 128- and 256-row tiles, split K; odd and whole sizes)
PRODUCTS = [(1, 1, 1), (1, 128, 128), (1, 100, 1000), (2, 33, 8), (16, 2049, 1280), (5, 700, 5000), (17, 96, 130), (33, 300, 1000),
            (64, 513, 640), (65, 300, 130), (128, 256, 128), (200, 256, 384), (256, 512, 1024), (333, 515, 2500),
            (700, 1000, 2048), (1025, 1300, 1152), (4100, 700, 520), (1, 40, 40000), (3, 17000, 300), (9, 70, 9001), (12, 50, 4608),
            (16, 40, 2600), (32, 129, 3100), (5, 5000, 300), (16, 8000, 520), (1, 8200, 300), (16, 12200, 130), (9, 15300, 260),
            (27, 15360, 130), (16, 20470, 300), (30, 20480, 200), (13, 21500, 300), (20, 24000, 130), (16, 32760, 130),
            (31, 30000, 130), (1, 32768, 200), (16, 2000, 14336), (29, 2000, 14336), (1, 50000, 130)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k", PRODUCTS)
def test_linear(dev, dtype, m, n, k):
    mx = _mx()
    x, w = _acts(m, k, dtype, m + n + k), _acts(n, k, torch.float32, n * k) * 0.05
    bias = _acts(1, n, dtype, 3)[0] if (m + n) % 2 else None
    p = mx.prepare_fp8_weight(w.to(dev))
    xv, wv = ob.rows(x)[0], ob.tiles(w)[0]
    b = None if bias is None else bias.to(dev)
    wide = m <= 16 or dtype == torch.float32
    y = mx.fp8_linear(x.to(dev), p, b)
    assert y.dtype == dtype
    check_product(y, xv, wv, bias, wide)
    # from the kept pair the same bits, wherever the two take the same kernel
    q, s = mx.quantize_fp8_block128(x.to(dev))
    assert torch.equal(mx.fp8_linear_prequantized(q, s, p, b, dtype), y)
    assert torch.equal(mx.fp8_linear_prequantized(q.contiguous(), s.contiguous(), p, b, dtype), y)


@pytest.mark.parametrize("out", DTYPES)
@pytest.mark.parametrize("m", [3, 80, 300])
def test_linear_output_types_and_shapes(dev, out, m):
    mx = _mx()
    x = _acts(2 * m, 520, torch.bfloat16, m).view(2, m, 520)
    w = _acts(130, 520, torch.float32, 9) * 0.05
    y = mx.fp8_linear(x.to(dev), mx.prepare_fp8_weight(w.to(dev)), out_dtype=out)
    assert y.shape == (2, m, 130) and y.dtype == out
    check_product(y.view(2 * m, 130), ob.rows(x.view(2 * m, 520))[0], ob.tiles(w)[0], None, 2 * m <= 16 or out == torch.float32)


def test_linear_of_no_rows(dev):
    mx = _mx()
    p = mx.prepare_fp8_weight(torch.randn(40, 256, device=dev))
    y = mx.fp8_linear(torch.zeros(0, 256, device=dev, dtype=torch.bfloat16), p)
    assert y.shape == (0, 40)
    q, s = mx.quantize_fp8_block128(torch.zeros(3, 0, 256, device=dev))
    assert q.shape == (3, 0, 256) and s.shape == (3, 0, 2)
    assert mx.dequantize_fp8_block128(q, s).shape == (3, 0, 256)
    assert mx.fp8_linear_prequantized(q, s, p).shape == (3, 0, 40)


@pytest.mark.parametrize("m", [1, 40, 100, 300])
def test_nan_stays_in_its_row(dev, m):
    """A NaN or an infinity of x makes its own row NaN and no other; one of the weight its own column."""
    mx = _mx()
    x, w = _acts(m, 384, torch.bfloat16, m), _acts(200, 384, torch.float32, 1) * 0.05
    x[m // 2, 7] = float("inf")
    y = mx.fp8_linear(x.to(dev), mx.prepare_fp8_weight(w.to(dev))).cpu()
    assert torch.equal(y.isnan().all(1), torch.arange(m) == m // 2) and torch.equal(y.isnan().any(1), y.isnan().all(1))
    x[m // 2, 7] = 1.0
    w[3, 100] = float("nan")
    y = mx.fp8_linear(x.to(dev), mx.prepare_fp8_weight(w.to(dev))).cpu()
    assert torch.equal(y.isnan().all(0), torch.arange(200) == 3) and torch.equal(y.isnan().any(0), y.isnan().all(0))


@pytest.mark.parametrize("m", [4, 100, 300])
def test_far_exponents(dev, m):
    """Blocks of very different magnitude in one row: each keeps its own scale."""
    mx = _mx()
    x = _acts(m, 640, torch.float32, 11, 0.0)
    x *= torch.exp2(torch.tensor([-40.0, 30.0, 0.0, -20.0, 10.0])).repeat_interleave(128)
    w = _acts(140, 640, torch.float32, 12, 0.0)
    w *= torch.exp2(torch.tensor([40.0, -30.0, 0.0, 20.0, -10.0])).repeat_interleave(128)
    y = mx.fp8_linear(x.to(dev), mx.prepare_fp8_weight(w.to(dev)))
    check_product(y, ob.rows(x)[0], ob.tiles(w)[0], None, True)


def test_two_streams_and_a_replayed_graph(dev):
    mx = _mx()
    p = mx.prepare_fp8_weight(_acts(900, 2048, torch.float32, 2).to(dev) * 0.05)
    xs = [_acts(m, 2048, torch.bfloat16, m).to(dev) for m in (1, 40, 130, 300)]
    want = [mx.fp8_linear(x, p) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = {}
    for i, st in enumerate(streams):
        with torch.cuda.stream(st):
            got[i] = [mx.fp8_linear(x, p) for x in xs]
    torch.cuda.synchronize()
    for i in got:
        for a, b in zip(got[i], want):
            assert torch.equal(a, b)
    static = [x.clone() for x in xs]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = [mx.fp8_linear(x, p) for x in static]
    for shift in (0.0, 1.0, -2.0):
        for x, s in zip(xs, static):
            s.copy_(x + shift)
        graph.replay()
        torch.cuda.synchronize()
        for s, o in zip(static, out):
            assert torch.equal(o, mx.fp8_linear(s, p))


def test_every_code_and_scale_byte(dev):
    """Pairs of other making: the value of all 256 codes under all 256 scale bytes (255 is NaN), restored and multiplied."""
    mx = _mx()
    q = torch.arange(256, dtype=torch.uint8).repeat(256, 1).view(torch.float8_e4m3fn)
    s = torch.arange(256, dtype=torch.uint8)[:, None].repeat(1, 2).view(torch.float8_e8m0fnu)
    ref = q.float().double() * s.float().double().repeat_interleave(128, 1)
    for dtype in DTYPES:
        got = mx.dequantize_fp8_block128(q.to(dev), s.to(dev), dtype)
        assert _same(got.cpu().double(), ref.to(dtype).double())
    # without the NaN codes: a product's row is NaN where its scale is, and exact for the scales that the quantizers give
    keep = torch.ones(256, dtype=torch.bool)
    keep[[127, 255]] = False
    z = q.view(torch.uint8).clone()
    z[:, ~keep] = 0
    p = mx.prepare_fp8_weight(torch.eye(256).to(dev))
    for first, last in ((0, 256), (100, 109), (220, 247), (250, 256)):
        rows = slice(first, last)
        y = mx.fp8_linear_prequantized(z[rows].view(torch.float8_e4m3fn).to(dev), s[rows].contiguous().to(dev), p, out_dtype=torch.float32)
        want = torch.where(keep[None, :], ref[rows], 0.0)
        want[torch.arange(first, last) == 255] = float("nan")
        byte = torch.arange(first, last)
        fair = ((byte >= 10) & (byte < 247)) | (byte == 255)  # (448 * 2^120 is beyond float32)
        assert _same(y.cpu().double()[fair], want.float().double()[fair])


@pytest.mark.parametrize("n,k", [(1, 1), (130, 205), (513, 1152), (300, 77)])
def test_weight_from_codes_of_any_layout(dev, n, k):
    """Codes and scales inside larger tensors, at odd offsets and strides, and transposed: the same form as from copies."""
    mx = _mx()
    g = _gen(n + k)
    nb, kb = -(-n // 128), -(-k // 128)
    big = torch.randint(0, 127, (n + 2, k + 10), generator=g, dtype=torch.uint8)
    sbig = torch.randint(100, 140, (nb + 1, kb + 3), generator=g, dtype=torch.uint8)
    codes, scales = big[1 : n + 1, 3 : k + 3], sbig[:nb, 1 : kb + 1]
    want_q = torch.zeros(n, kb * 128, dtype=torch.uint8)
    want_q[:, :k] = codes
    want_t = torch.zeros(k, nb * 128, dtype=torch.uint8)
    want_t[:, :n] = codes.t()

    def dev8(t, dtype):
        return t.to(dev).view(dtype)

    f8, e8 = torch.float8_e4m3fn, torch.float8_e8m0fnu
    for w, s in ((dev8(big, f8)[1 : n + 1, 3 : k + 3], dev8(sbig, e8)[:nb, 1 : kb + 1]),
                 (dev8(codes.t().contiguous(), f8).t(), dev8(scales.t().contiguous(), e8).t())):
        for transposed in (True, False):
            p = mx.prepare_fp8_weight(w, s, transposed)
            assert torch.equal(p.q.cpu().view(torch.uint8), want_q)
            assert torch.equal(p.scale.cpu().view(torch.uint8)[:, :kb], scales)
            if transposed:
                assert torch.equal(p.qt.cpu().view(torch.uint8), want_t)
                assert torch.equal(p.scale_t.cpu().view(torch.uint8)[:, :nb], scales.t())
            else:
                assert p.qt is None and p.scale_t is None


def test_restoring_more_than_one_launch_counts(dev):
    """2^31 pieces of 16 bytes and some: what can be put away can be taken out."""
    mx = _mx()
    m = 2**26 + 3
    q = torch.zeros(m, 128, dtype=torch.uint8, device=dev)
    s = torch.full((m, 1), 127, dtype=torch.uint8, device=dev)
    at = torch.tensor([0, 1, 2**25, 2**26 - 2050, 2**26 - 2049, 2**26 - 2048, 2**26 - 1, 2**26, m - 1], device=dev)
    q[at, 7] = 0x40  # 2
    s[at, 0] = 130
    out = mx.dequantize_fp8_block128(q.view(torch.float8_e4m3fn), s.view(torch.float8_e8m0fnu), torch.float32)
    assert bool((out[at, 7] == 16).all())
    assert sum(int(torch.count_nonzero(part)) for part in out.split(2**24)) == at.numel()


# ---------------------------------------------------------------------------------------
# the scaled matrix instruction: 16-bit results of more than 16 rows
# ---------------------------------------------------------------------------------------
# Its cuts: 64 addends, each by at most 2^-13 of the largest. Where their signs are independent, an element's error has at
# most the variance 64 (2^-13 max|p|)^2 per 64 columns, and the last rounding, uniform within half a step u, u^2 / 3 y^2.

HALVES = [torch.bfloat16, torch.float16]


def _cut_variance(xv, wv):
    """Sum over 64-long pieces of 64 (2^-13 max|x w|)^2, [M, N]."""
    out = torch.zeros(xv.shape[0], wv.shape[0], dtype=torch.float64)
    for k in range(0, xv.shape[1], 64):
        p = (xv[:, None, k : k + 64].abs() * wv[None, :, k : k + 64].abs()).amax(-1)
        out += 64 * (2.0**-13 * p) ** 2
    return out


def _check_norm_of_cuts(y, xv, wv):
    ref = xv @ wv.t()
    u = _half_step(y.dtype)
    err = float((y.double().cpu() - ref).square().sum())
    assert err <= float(u * u / 3 * ref.square().sum() + _cut_variance(xv, wv).sum()) * (1 + 2.0**-6)


@pytest.mark.parametrize("out", HALVES)
@pytest.mark.parametrize("m", [40, 100, 300])
def test_each_block_has_its_own_scale(dev, out, m):
    """Rows of one block that is not zero, at far exponents of the row's and the tile's own: the result is that block's product
    alone, so a scale taken from another stage, row or tile shows whole."""
    mx = _mx()
    n, kb = 300, 11
    g = _gen(m)
    x = torch.randn(m, kb, 128, generator=g)
    e = torch.randint(-50, 51, (m, kb), generator=g)
    f = torch.randint(-50, 51, (-(-n // 128), kb), generator=g)
    keep = torch.arange(m)[:, None] % kb == torch.arange(kb)
    # (the tile's exponent is undone by the row's, but for up to 2^5: results stay in float16's range)
    x = torch.ldexp(x, e[..., None]) * keep[..., None]
    w = torch.ldexp(torch.randn(n, kb, 128, generator=g), f.repeat_interleave(128, 0)[:n][..., None])
    for tile in range(f.shape[0]):  # one column tile at a time: its exponents undone
        rows = slice(tile * 128, min(n, tile * 128 + 128))
        scale = torch.ldexp(torch.ones(()), (-(e + f[tile]) - 4 + (torch.arange(m)[:, None] % 6))[..., None])
        xt = (x * scale).view(m, -1)
        y = mx.fp8_linear(xt.to(dev), mx.prepare_fp8_weight(w.view(n, -1).to(dev)), out_dtype=out).cpu()
        xv, wv = ob.rows(xt)[0], ob.tiles(w.view(n, -1))[0][rows]
        check_product(y[:, rows], xv, wv, None, False)
        _check_norm_of_cuts(y[:, rows], xv, wv)


@pytest.mark.parametrize("out", HALVES)
def test_every_code_and_scale_byte_of_the_scaled_instruction(dev, out):
    """All codes under all scale bytes (255: NaN) of an activation, and of a weight, times one."""
    mx = _mx()
    q = torch.arange(256, dtype=torch.uint8).repeat(256, 1)
    q[:, [127, 255]] = 0
    s = torch.arange(256, dtype=torch.uint8)[:, None].repeat(1, 2)
    byte = torch.arange(256)
    ref = ob.e4m3_table()[q.long()] * torch.ldexp(torch.ones((), dtype=torch.float64), byte - 127)[:, None]
    ref[255] = float("nan")
    fair = ((byte >= 10) & (byte < 247)) | (byte == 255)  # (the scales that the quantizers give of finite values in range)
    p = mx.prepare_fp8_weight(torch.eye(256).to(dev))
    y = mx.fp8_linear_prequantized(q.view(torch.float8_e4m3fn).to(dev), s.view(torch.float8_e8m0fnu).to(dev), p, out_dtype=out)
    assert _same(y.cpu().double()[fair], ref.to(out).double()[fair])
    # a weight of three tiles of equal rows, each under its byte: row j of the identity picks code j
    xq, xs = mx.quantize_fp8_block128(torch.eye(128).to(dev))
    codes = torch.arange(128, dtype=torch.uint8)
    codes[127] = 0
    for first in range(10, 241, 33):
        b = torch.tensor([first, 255, first + 6], dtype=torch.uint8)
        w = mx.prepare_fp8_weight(codes.repeat(384, 1).view(torch.float8_e4m3fn).to(dev), b[:, None].view(torch.float8_e8m0fnu).to(dev))
        y = mx.fp8_linear_prequantized(xq, xs, w, out_dtype=out).cpu().double()
        for t in range(3):
            v = ob.e4m3_table()[codes.long()] * (float("nan") if t == 1 else 2.0 ** (int(b[t]) - 127))
            assert _same(y[:, t * 128 : t * 128 + 128], v.to(out).double()[:, None].expand(128, 128))


@pytest.mark.parametrize("out", HALVES)
@pytest.mark.parametrize("m,n,k", [(40, 96, 1152), (130, 200, 2000)])
def test_outlier_channels(dev, out, m, n, k):
    """One channel in 200 twenty times larger, as transformers' activations have them."""
    mx = _mx()
    g = _gen(k)
    x = torch.randn(m, k, generator=g)
    x[:, torch.randperm(k, generator=g)[: k // 200]] *= 20
    w = torch.randn(n, k, generator=g) * 0.02
    y = mx.fp8_linear(x.to(out).to(dev), mx.prepare_fp8_weight(w.to(dev)))
    xv, wv = ob.rows(x.to(out))[0], ob.tiles(w)[0]
    check_product(y, xv, wv, None, False)
    _check_norm_of_cuts(y, xv, wv)


@pytest.mark.parametrize("out", DTYPES)
@pytest.mark.parametrize("m", [3, 100, 300])
def test_small_addends_of_one_sign(dev, out, m):
    """The worst case of the scaled instruction's cuts: beside one product, 63 of its own sign just below 2^-13 of it. Up to
    16 rows and float32 results have them; 16-bit results of more rows are within 64 cuts of 2^-13 of the largest."""
    mx = _mx()
    x = torch.full((m, 640), 1.875 * 2.0**-6)
    x[:, ::64] = 256.0
    w = torch.ones(130, 640)
    wide = m <= 16 or out == torch.float32
    y = mx.fp8_linear(x.to(out).to(dev), mx.prepare_fp8_weight(w.to(dev)), out_dtype=out)
    xv, wv = ob.rows(x)[0], ob.tiles(w)[0]
    assert torch.equal(xv, x.double())
    check_product(y, xv, wv, None, wide)


@pytest.mark.parametrize("out", HALVES)
@pytest.mark.parametrize("m,n,k", [(5, 40, 300), (31, 40, 300), (33, 300, 1000), (200, 256, 384), (333, 515, 2500), (1025, 1300, 1152),
                                   (4100, 700, 520), (100, 130, 20000)])
def test_full_sums(dev, out, m, n, k):
    """16-bit results with every addend: the float32 result rounded, within float32's own bounds."""
    mx = _mx()
    x, w, bias = _acts(m, k, out, m + n), _acts(n, k, torch.float32, n * k) * 0.05, _acts(1, n, out, 3)[0]
    p = mx.prepare_fp8_weight(w.to(dev))
    y = mx.fp8_linear(x.to(dev), p, bias.to(dev), full_sums=True)
    assert y.dtype == out
    check_product(y, ob.rows(x)[0], ob.tiles(w)[0], bias, True)
    assert torch.equal(y, mx.fp8_linear(x.to(dev), p, bias.to(dev), out_dtype=torch.float32).to(out))
    q, s = mx.quantize_fp8_block128(x.to(dev))
    assert torch.equal(mx.fp8_linear_prequantized(q, s, p, bias.to(dev), out, full_sums=True), y)


@pytest.mark.parametrize("out", HALVES)
@pytest.mark.parametrize("m", [100, 300])
def test_small_addends_of_one_sign_in_full_sums(dev, out, m):
    mx = _mx()
    x = torch.full((m, 640), 1.875 * 2.0**-6)
    x[:, ::64] = 256.0
    w = torch.ones(130, 640)
    y = mx.fp8_linear(x.to(out).to(dev), mx.prepare_fp8_weight(w.to(dev)), full_sums=True)
    check_product(y, x.double(), ob.tiles(w)[0], None, True)
