"""The rms norm on the GPU against its definition (oracle/mxfp4_block.py, oracle/fp8_block.py).

The forward pass is held to the bit: given the kernel's own rstd, y is two float32 multiplications and one rounding; rstd is
half a step of float32 off the float64 value (2^-24, and 2^-40 for the estimate's refinement and the order of the float64
sum). Codes are those of that y, bit for bit.

The backward pass sums in float32. c = E[g xh] has at most D + 6 roundings of 2^-24 of its largest partial sum, at most
A = r^2 E|g x|; dx has six more, each of at most the largest of its three terms: |error| <= u |dx| + 2^-24 ((D + 8) |x| A + 6
(|r g| + |x| A + |ds|)). dw has M + 4 roundings of at most the sum of magnitudes of its column.
"""

from __future__ import annotations

import pytest
import torch

from oracle import fp8_block as o8
from oracle import mxfp4_block as ob

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]
NORMS = [(1, 1), (1, 5120), (3, 7), (5, 8), (4, 100), (2, 511), (9, 512), (3, 513), (65, 1003), (7, 1024), (5, 1500), (4, 2048), (3, 3001),
         (130, 4096), (2, 5376), (3, 6145), (2, 8200), (3, 12288), (2, 20480), (2, 24575), (2, 24576)]
# A head's columns: rows that share a wave, the last of a workgroup's missing, runs of eight that end in every place.
NARROW = [(1, 64), (15, 128), (17, 128), (1000, 128), (33, 127), (31, 121), (2, 129), (65, 200), (9, 256), (1003, 256), (5, 257), (18, 9),
          (35, 2), (4, 130), (7, 252), (5000, 96)]


def _mx():
    import mx_qlinear

    return mx_qlinear


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _acts(m, d, dtype, seed, spread=1.0):
    g = _gen(seed)
    return (torch.randn(m, d, generator=g) * torch.exp(spread * torch.randn(m, 1, generator=g))).to(dtype)


def _weight(d, dtype, seed):
    return (1 + 0.3 * torch.randn(d, generator=_gen(seed))).to(dtype)


def check_rstd(rstd, s, eps):
    ref = 1.0 / (s.double().square().mean(1) + eps).sqrt()
    assert bool(((rstd.double().cpu() - ref).abs() <= (2.0**-24 + 2.0**-40) * ref).all())


def check_codes8(q, s, y):
    want, e = o8.rows(y)
    assert torch.equal(s.cpu().contiguous().view(torch.uint8).int() - 127, e)
    got = o8.values(q, s)
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(0.0), want.nan_to_num(0.0))


def check_codes4(q, s, y):
    _, b, codes = ob.rows(y)
    assert torch.equal(s.cpu().contiguous().view(torch.uint8).int(), b)
    assert torch.equal(q.cpu().contiguous().view(torch.uint8), ob.pack(codes))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,d", NORMS + NARROW)
def test_forward(dev, dtype, m, d):
    mx = _mx()
    x, r, w = _acts(m, d, dtype, m + d, 2.0), _acts(m, d, dtype, m + d + 1, 2.0), _weight(d, dtype, d)
    on = (x.to(dev), w.to(dev), 1e-6)
    for residual in (None, r):
        s = x if residual is None else (x.float() + r.float()).to(dtype)
        kw = {"residual": None if residual is None else r.to(dev), "return_rstd": True}
        y, *rest = mx.rms_norm(*on, **kw)
        rstd = rest[-1]
        check_rstd(rstd, s, 1e-6)
        want = ob.normed(s, rstd.cpu(), w)
        assert y.dtype == dtype and torch.equal(y.cpu(), want.to(dtype))
        q8, s8, *rest8 = mx.rms_norm_quantize_fp8(*on, **kw)
        check_codes8(q8, s8, want)
        q4, s4, *rest4 = mx.rms_norm_quantize_mxfp4(*on, **kw)
        check_codes4(q4, s4, want)
        for other in (rest, rest8, rest4):
            assert torch.equal(other[-1], rstd) and len(other) == (1 if residual is None else 2)
            if residual is not None:
                assert torch.equal(other[0].cpu(), s)


@pytest.mark.parametrize("dtype", DTYPES)
def test_layouts_and_parameters(dev, dtype):
    mx = _mx()
    base, rbase = _acts(24, 700, dtype, 1), _acts(24, 650, dtype, 2)
    on, ron = base.to(dev), rbase.to(dev)
    for d, a, b in ((600, 3, 50), (608, 8, 16), (33, 1, 2)):
        x, r = base[:, a:a + d], rbase[:, b:b + d] if d <= 600 else rbase[:, 16:624]
        y, s, rstd = mx.rms_norm(on[:, a:a + d], None, 1e-5, residual=(ron[:, b:b + d] if d <= 600 else ron[:, 16:624]), return_rstd=True)
        want = (x.float() + r.float()).to(dtype)
        assert torch.equal(s.cpu(), want) and torch.equal(y.cpu(), ob.normed(want, rstd.cpu(), None).to(dtype))
    w = _weight(700, torch.float32, 3)
    for weight in (w, w.to(torch.bfloat16), w.half()):  # (of another type than x: as float32)
        y, rstd = mx.rms_norm(on, weight.to(dev), return_rstd=True)
        assert torch.equal(y.cpu(), ob.normed(base, rstd.cpu(), weight).to(dtype))
    y, s, rstd = mx.rms_norm(on.view(2, 3, 4, 700), residual=on.view(2, 3, 4, 700), return_rstd=True)  # (x is its own residual)
    assert y.shape == s.shape == (2, 3, 4, 700) and rstd.shape == (2, 3, 4)
    assert torch.equal(s.cpu().view(24, 700), (base.float() * 2).to(dtype))
    q, sc, s, rstd = mx.rms_norm_quantize_mxfp4(on.view(2, 12, 700)[1, 5], residual=on[0], return_rstd=True)
    assert q.shape == (350,) and sc.shape == (22,) and s.shape == (700,) and rstd.shape == ()
    q, sc = mx.rms_norm_quantize_fp8(on.view(2, 12, 700))
    assert q.shape == (2, 12, 700) and sc.shape == (2, 12, 6)
    assert mx.rms_norm(on[:0]).shape == (0, 700)
    assert [t.shape for t in mx.rms_norm_quantize_mxfp4(on[:0], residual=on[:0])] == [(0, 350), (0, 22), (0, 700)]
    strided = mx.rms_norm(on[::3], return_rstd=True)
    assert torch.equal(strided[0].cpu(), ob.normed(base[::3], strided[1].cpu(), None).to(dtype))
    copied = mx.rms_norm(on.t(), return_rstd=True)
    assert torch.equal(copied[0].cpu(), ob.normed(base.t(), copied[1].cpu(), None).to(dtype))


@pytest.mark.parametrize("dtype", DTYPES)
def test_far_rows(dev, dtype):
    """Zeros with and without eps, the largest and smallest magnitudes, NaN and infinities: as the formula in torch has them."""
    mx = _mx()
    top = torch.finfo(dtype).max
    x = torch.zeros(9, 300, dtype=torch.float64)
    x[1, :] = top
    x[2, 7] = top
    x[3, :] = torch.finfo(dtype).smallest_normal
    x[4, 5] = float("nan")
    x[5, 5], x[5, 6] = float("inf"), 2.0
    x[6, :] = -1.0
    x[7, 299] = float("-inf")
    x[8, 0] = 1.0
    x = x.to(dtype)
    for eps in (0.0, 1e-6):
        ref = 1.0 / (x.double().square().mean(1) + torch.tensor(eps, dtype=torch.float32).double()).sqrt()
        y, rstd = mx.rms_norm(x.to(dev), None, eps, return_rstd=True)
        got = rstd.cpu().double()
        fine = torch.isfinite(ref) & (ref < 3e38)
        assert torch.equal(torch.isfinite(got), fine) and torch.equal(got.isnan(), ref.isnan())
        assert bool(((got - ref).abs() <= (2.0**-24 + 2.0**-40) * ref + 2.0**-149)[fine].all())
        want = ob.normed(x, rstd.cpu(), None).to(dtype)
        assert torch.equal(y.cpu().isnan(), want.isnan()) and torch.equal(y.cpu().nan_to_num(0.0), want.nan_to_num(0.0))
        check_codes8(*mx.rms_norm_quantize_fp8(x.to(dev), None, eps), ob.normed(x, rstd.cpu(), None))
        check_codes4(*mx.rms_norm_quantize_mxfp4(x.to(dev), None, eps), ob.normed(x, rstd.cpu(), None))


# ---------------------------------------------------------------------------------------
# gradients
# ---------------------------------------------------------------------------------------

def check_backward(dx, dw, dy, s, rstd, weight, dsum):
    ref, refw = ob.rms_norm_backward(dy, s, rstd, weight, dsum)
    u, (m, d) = torch.finfo(dx.dtype).eps / 2, dy.shape
    x, r = s.double().abs(), rstd.double()[:, None]
    g = dy.double().abs() * (1 if weight is None else weight.double().abs())
    a = r * r * (g * x).mean(1, keepdim=True)
    terms = r * g + x * a + (0 if dsum is None else dsum.double().abs())
    bound = u * ref.abs() + 2.0**-24 * ((d + 8) * x * a + 6 * terms) + torch.finfo(dx.dtype).tiny
    err = (dx.double().cpu() - ref).abs()
    assert bool((err <= bound * (1 + u)).all()), f"worst {float((err / bound).max())} of the bound"
    if dw is not None:
        bound = 2.0**-24 * (m + 4) * (dy.double().abs() * x * r).sum(0) + 2.0**-140
        assert bool(((dw.double().cpu() - refw).abs() <= bound).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,d", [*NORMS, *NARROW, (700, 64), (2100, 513), (600, 1536)])
def test_backward(dev, dtype, m, d):
    mx = _mx()
    x, w, dy, ds = _acts(m, d, dtype, m + d), _weight(d, dtype, d), _acts(m, d, dtype, m + d + 2) * 0.1, _acts(m, d, dtype, m + d + 3) * 0.1
    rstd = (x.double().square().mean(1) + 1e-6).rsqrt().float()
    for dsum in (None, ds):
        on = None if dsum is None else ds.to(dev)
        dx, dw = mx.rms_norm_backward(dy.to(dev), x.to(dev), rstd.to(dev), w.to(dev), on)
        assert dx.dtype == dtype and dw.dtype == torch.float32
        check_backward(dx, dw, dy, x, rstd, w, dsum)
        again, none = mx.rms_norm_backward(dy.to(dev), x.to(dev), rstd.to(dev), w.to(dev), on, needs_params=False)
        assert none is None and torch.equal(again, dx)
        q, s = mx.quantize_fp8_block128(x.to(dev))
        kept = o8.values(q, s)
        dx, dw = mx.rms_norm_backward(dy.to(dev), (q, s), rstd.to(dev), w.to(dev), on)
        check_backward(dx, dw, dy, kept, rstd, w, dsum)
        assert all(torch.equal(a, b) for a, b in zip(mx.rms_norm_backward(dy.to(dev), (q, s), rstd.to(dev), w.to(dev), on), (dx, dw)))


@pytest.mark.parametrize("dtype", DTYPES)
def test_backward_layouts(dev, dtype):
    mx = _mx()
    base = _acts(30, 900, dtype, 1)
    on = base.to(dev)
    dy, x, ds = base[:, 1:601], base[:, 200:800], base[::1, 299:899]
    rstd = (x.double().square().mean(1) + 1e-6).rsqrt().float()
    w = _weight(600, torch.float32, 2)
    dx, dw = mx.rms_norm_backward(on[:, 1:601], on[:, 200:800], rstd.to(dev), w.to(dev), on[:, 299:899])
    check_backward(dx, dw, dy, x, rstd, w, ds)
    dx, dw = mx.rms_norm_backward(on[:, 1:601].unflatten(0, (5, 6)), on[:, 200:800].unflatten(0, (5, 6)), rstd.view(5, 6).to(dev))
    assert dx.shape == (5, 6, 600)
    check_backward(dx.flatten(0, 1), dw, dy, x, rstd, None, None)
    q, s = mx.quantize_fp8_block128(on)
    far = (q[:, 128:728], s[:, 1:6])
    xk = o8.values(q, s)[:, 128:728]
    dx, dw = mx.rms_norm_backward(on[:, 1:601], far, rstd.to(dev), w.to(dev))
    check_backward(dx, dw, dy, xk, rstd, w, None)
    dx, dw = mx.rms_norm_backward(on[:0], on[:0], rstd[:0].to(dev))
    assert dx.shape == (0, 900) and bool((dw == 0).all())
    dx, dw = mx.rms_norm_backward(on[:1, :77].expand(4, 77), on[:4, :77], rstd[:4].to(dev))
    check_backward(dx, dw, base[:1, :77].expand(4, 77), base[:4, :77], rstd[:4], None, None)


def check_far_backward(dx, dw, dy, s, rstd, weight, dsum, steps):
    """dx = r g - (xh r) c + ds with c = E[g xh], whose magnitudes are T1 = |r g|, T2 = |xh| r E|g xh| and |ds|. The sum of c has at
    most D roundings of its partial sums, each at most E|g xh|; six more steps (xh, g, the three products, the sum) are each
    half a step of float32 of the terms; ``steps`` are those of an rstd that is not the kernel's own."""
    ref, refw = ob.rms_norm_backward(dy, s, rstd, weight, dsum)
    u, (m, d) = torch.finfo(dx.dtype).eps / 2, dy.shape
    r = rstd.double()[:, None]
    xh = s.double().abs() * r
    g = dy.double().abs() * (1 if weight is None else weight.double().abs())
    t2 = xh * r * (g * xh).mean(1, keepdim=True)
    terms = r * g + t2 + (0 if dsum is None else dsum.double().abs())
    bound = u * ref.abs() + 2.0**-24 * ((d + 8) * t2 + (6 + steps) * terms) + torch.finfo(dx.dtype).tiny
    err = (dx.double().cpu() - ref).abs()
    assert bool((err <= bound * (1 + u)).all()), f"rows at worst {(err / bound).amax(1).tolist()} of the bound"
    if dw is not None:
        bound = 2.0**-24 * (m + 4) * (dy.double().abs() * xh).sum(0) + 2.0**-140
        assert bool(((dw.double().cpu() - refw).abs() <= bound).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("d", [5, 128, 200, 300, 1003, 5120, 9000, 20480])
def test_backward_of_far_rows(dev, dtype, d):
    """Rows of every magnitude that the forward pass takes, one of each in a tensor, by themselves and kept in 8 bits: rstd
    squared is beyond float32 in half of them, the gradient is not. dy has a share along the row, so that the term with
    rstd squared is of the size of the other."""
    mx = _mx()
    sizes = torch.tensor([1e-30, 1e-20, 1e-19, 1e-10, 1.0, 1e10, 1e19, 1e20, 1e22, 1e24, 1e30, 1e36])[:, None]
    unit = _acts(12, d, torch.float32, d, 0.0)
    x, w = (unit * sizes).to(dtype), _weight(d, dtype, d + 1)
    dy = (0.1 * _acts(12, d, torch.float32, d + 2, 0.0) + 0.2 * unit).to(dtype)
    rstd = x.double().square().mean(1).rsqrt().float()
    for ds in (None, (dy.float() * rstd[:, None]).to(dtype)):
        on = None if ds is None else ds.to(dev)
        dx, dw = mx.rms_norm_backward(dy.to(dev), x.to(dev), rstd.to(dev), w.to(dev), on)
        check_far_backward(dx, dw, dy, x, rstd, w, ds, 0)
        q, s = mx.quantize_fp8_block128(x.to(dev))
        dx, dw = mx.rms_norm_backward(dy.to(dev), (q, s), rstd.to(dev), w.to(dev), on)
        check_far_backward(dx, dw, dy, o8.values(q, s), rstd, w, ds, 0)
    # through the module: its own rstd is one rounding off, a step of float32 in T1 and three in T2
    for keep in (False, True):
        norm = mx.RMSNorm(d, 0.0, keep_fp8=keep, device=dev, dtype=dtype)
        norm.weight.data.copy_(w)
        xx = x.to(dev).requires_grad_()
        norm(xx).backward(dy.to(dev))
        kept = o8.values(*mx.quantize_fp8_block128(x.to(dev))) if keep else x
        check_far_backward(xx.grad, None, dy, kept, rstd, w, None, 8)


def test_backward_against_differences(dev):
    """float32 central differences of sum(y dy) + sum(s ds): steps of 2^-7 leave 2^-14 |x| of curvature and 2^-24 / 2^-7 of
    rounding, each times the row's sums of magnitudes."""
    mx = _mx()
    d = 96
    x, r = _acts(3, d, torch.float32, 1, 0.0), _acts(3, d, torch.float32, 2, 0.0)
    w, dy, ds = _weight(d, torch.float32, 3), _acts(3, d, torch.float32, 4, 0.0), _acts(3, d, torch.float32, 5, 0.0)

    def loss(xx):
        y, s = mx.rms_norm(xx.to(dev), w.to(dev), 1e-6, residual=r.to(dev))
        return (y.cpu().double() * dy.double()).sum(1) + (s.cpu().double() * ds.double()).sum(1)

    _, s, rstd = mx.rms_norm(x.to(dev), w.to(dev), 1e-6, residual=r.to(dev), return_rstd=True)
    dx, _ = mx.rms_norm_backward(dy.to(dev), s, rstd, w.to(dev), ds.to(dev))
    h = 2.0**-7
    size = (dy.abs() * w.abs() * s.cpu().abs()).sum(1).double() + (s.cpu().abs() * ds.abs()).sum(1).double()
    for j in (0, 1, 50, 95):
        up, down = x.clone(), x.clone()
        up[:, j] += h
        down[:, j] -= h
        step = (up[:, j].double() - down[:, j].double())
        diff = (loss(up) - loss(down)) / step
        assert bool(((dx[:, j].cpu().double() - diff).abs() <= 2.0**-13 * size).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("keep", [False, True])
@pytest.mark.parametrize("residual", [False, True])
def test_module(dev, dtype, keep, residual):
    mx = _mx()
    m, d = 37, 520
    x, r, w = _acts(m, d, dtype, 1), _acts(m, d, dtype, 2), _weight(d, dtype, 3)
    dy, ds = _acts(m, d, dtype, 4), _acts(m, d, dtype, 5)
    norm = mx.RMSNorm(d, 1e-6, keep_fp8=keep, device=dev, dtype=dtype)
    norm.weight.data.copy_(w)
    xx = x.to(dev).requires_grad_()
    rr = r.to(dev).requires_grad_()
    out = norm(xx, rr) if residual else norm(xx)
    if residual:
        torch.autograd.backward(out, (dy.to(dev), ds.to(dev)))
    else:
        out.backward(dy.to(dev))
    s = (x.float() + r.float()).to(dtype) if residual else x
    rstd = (s.double().square().mean(1) + 1e-6).rsqrt().float()
    if keep:
        s = o8.values(*mx.quantize_fp8_block128(s.to(dev)))
    # (rstd may be one rounding off the kernel's: four more steps of float32 in all)
    check_backward(xx.grad, None, dy, s, rstd, w, ds if residual else None)
    if residual:
        assert torch.equal(rr.grad, xx.grad)
    refw = ob.rms_norm_backward(dy, s, rstd, w)[1]
    bound = (torch.finfo(dtype).eps / 2) * refw.abs() + 2.0**-24 * (m + 8) * (dy.double().abs() * s.double().abs() * rstd.double()[:, None]).sum(0)
    assert bool(((norm.weight.grad.double().cpu() - refw).abs() <= bound * 1.01).all())
    with torch.no_grad():
        plain = norm(x.to(dev), r.to(dev)) if residual else norm(x.to(dev))
    for a, b in zip(plain if residual else (plain,), out if residual else (out,)):
        assert torch.equal(a, b)


def test_unused_outputs(dev):
    """Only the sum used, only the norm used, nothing needing a gradient."""
    mx = _mx()
    norm = mx.RMSNorm(64, device=dev)
    x, r = (torch.randn(5, 64, device=dev, requires_grad=True) for _ in range(2))
    _, s = norm(x, r)
    s.sum().backward()
    assert bool((x.grad == 1).all()) and bool((r.grad == 1).all()) and norm.weight.grad is None
    x.grad = r.grad = None
    y, _ = norm(x, r.detach())
    y.sum().backward()
    assert r.grad is None and x.grad.shape == (5, 64) and norm.weight.grad is not None
    norm.weight.requires_grad_(False)
    y, s = norm(x.detach(), r.detach())
    assert not y.requires_grad and not s.requires_grad


# ---------------------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m", [1, 16, 40, 300])
def test_norms_feed_the_layers(dev, dtype, m):
    """norm -> codes -> product equals norm -> float32 -> quantizer -> product, for both layers."""
    mx = _mx()
    d, n = 640, 96
    x, r, w = _acts(m, d, dtype, 1).to(dev), _acts(m, d, dtype, 2).to(dev), _weight(d, dtype, 3).to(dev)
    weight = _acts(n, d, torch.bfloat16, 4).to(dev)
    w4, w8 = mx.prepare_mxfp4_weight(weight), mx.prepare_fp8_weight(weight)
    q, s, total, rstd = mx.rms_norm_quantize_mxfp4(x, w, 1e-6, residual=r, return_rstd=True)
    y = ob.normed(total.cpu(), rstd.cpu(), w.cpu()).to(dev)
    assert torch.equal(mx.mxfp4_linear_prequantized(q, s, w4, out_dtype=dtype),
                       mx.mxfp4_linear_prequantized(*mx.quantize_mxfp4(y), w4, out_dtype=dtype))
    q, s, *_ = mx.rms_norm_quantize_fp8(x, w, 1e-6, residual=r)
    assert torch.equal(mx.fp8_linear_prequantized(q, s, w8, out_dtype=dtype),
                       mx.fp8_linear_prequantized(*mx.quantize_fp8_block128(y), w8, out_dtype=dtype))


def test_block_trained_around_a_frozen_layer(dev):
    """Two pre-norm layers on a residual stream: every gradient against float64 autograd of the held values; bfloat16 path,
    so each of the roundings of the stream (2^-9 of it a layer) is let through."""
    mx = _mx()
    m, d = 60, 256
    w = [_acts(d, d, torch.float32, i, 0.0) * d**-0.5 for i in (1, 2)]
    norms = [mx.RMSNorm(d, 1e-6, device=dev) for _ in range(2)]
    layers = [mx.Mxfp4Linear.from_weight(t.to(dev), torch.zeros(d, device=dev)) for t in w]
    x = _acts(m, d, torch.float32, 5, 0.0).to(dev).requires_grad_()
    y, s = norms[0](x, torch.zeros_like(x))
    y, s = norms[1](layers[0](y), s)
    out = layers[1](y)
    dy = _acts(m, d, torch.float32, 6, 0.0).to(dev)
    torch.autograd.backward((out, s), (dy, 0.1 * dy))
    # float64, the quantizers passing gradients through
    wv = [ob.rows(t)[0] for t in w]
    hold = lambda t: t + (ob.rows(t.detach())[0] - t.detach())  # noqa: E731
    norm64 = lambda t, g: t * (t.square().mean(1, keepdim=True) + 1e-6).rsqrt() * g  # noqa: E731
    x64 = x.detach().cpu().double().requires_grad_()
    g64 = [torch.ones(d, dtype=torch.float64, requires_grad=True) for _ in range(2)]
    b64 = [torch.zeros(d, dtype=torch.float64, requires_grad=True) for _ in range(2)]
    s64 = x64 + hold(norm64(x64, g64[0])) @ wv[0].t() + b64[0]
    out64 = hold(norm64(s64, g64[1])) @ wv[1].t() + b64[1]
    torch.autograd.backward((out64, s64), (dy.cpu().double(), 0.1 * dy.cpu().double()))
    # float32 throughout: a code at a border may fall the other way (1 in 2^18 of them, by a sixth of its value): 2^-9 in norm
    close = lambda a, b: float((a.detach().cpu().double() - b).norm() / b.norm()) <= 2.0**-9  # noqa: E731
    assert close(out, out64.detach()) and close(x.grad, x64.grad)
    for i in range(2):
        assert close(norms[i].weight.grad, g64[i].grad) and close(layers[i].bias.grad, b64[i].grad)


@pytest.mark.parametrize("m,d", [(1, 5120), (50, 300), (600, 1536)])
def test_captured_and_replayed(dev, m, d):
    mx = _mx()
    x, r, dy = (_acts(m, d, torch.bfloat16, i).to(dev) for i in (1, 2, 3))
    w = _weight(d, torch.bfloat16, 4).to(dev)

    def step():
        y, s, rstd = mx.rms_norm(x, w, residual=r, return_rstd=True)
        q4, s4 = mx.rms_norm_quantize_mxfp4(x, w)
        q8, s8 = mx.rms_norm_quantize_fp8(x, w)
        return (y, s, rstd, q4.view(torch.uint8), s4.view(torch.uint8), q8.view(torch.uint8), s8.view(torch.uint8),
                *mx.rms_norm_backward(dy, s, rstd, w, dy), *mx.rms_norm_backward(dy, (q8, s8), rstd, w))

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for seed in range(3):
        for i, t in enumerate((x, r, dy)):
            t.copy_(_acts(m, d, torch.bfloat16, 10 * seed + i))
        want = step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_module_is_not_captured(dev):
    mx = _mx()
    norm = mx.RMSNorm(256, device=dev)
    x = torch.randn(32, 256, device=dev)
    with torch.no_grad():
        want = norm(x)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="not captured"):
            norm(x)
        with torch.no_grad():
            y = norm(x)
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want)


@pytest.mark.parametrize("m,d", [(210_000, 20_480), (33_600_000, 128)])
def test_more_than_2_to_the_32_elements(dev, m, d):
    """Rows on both sides of every power of two that an offset could be cut at."""
    mx = _mx()
    x = torch.empty(m, d, dtype=torch.bfloat16, device=dev)
    for i in range(0, m, m // 5):
        x[i:i + m // 5].normal_()
    at = sorted({0, m - 1, *(min(m - 1, 2**p // d + e) for p in (29, 30, 31, 32) for e in (-1, 0, 1))})
    at = torch.tensor([i for i in at if 0 <= i < m])
    w = _weight(d, torch.bfloat16, 3)
    y, s, rstd = mx.rms_norm(x, w.to(dev), 1e-6, residual=x, return_rstd=True)
    few = (2 * x[at.to(dev)].float()).to(torch.bfloat16).cpu()
    assert torch.equal(s[at.to(dev)].cpu(), few)
    r = rstd[at.to(dev)].cpu()
    check_rstd(r, few, 1e-6)
    want = ob.normed(few, r, w)
    assert torch.equal(y[at.to(dev)].cpu(), want.to(torch.bfloat16))
    del y
    q, sc = mx.rms_norm_quantize_mxfp4(x, w.to(dev), 1e-6, residual=x)[:2]
    check_codes4(q.view(torch.uint8)[at.to(dev)].view(torch.float4_e2m1fn_x2), sc.view(torch.uint8)[at.to(dev)].view(torch.float8_e8m0fnu),
                 want)
    del q, sc
    dx, dw = mx.rms_norm_backward(x, s, rstd, w.to(dev), x)
    check_backward(dx[at.to(dev)], None, x[at.to(dev)].cpu(), few, r, w, x[at.to(dev)].cpu())
    total, size = torch.zeros(d, dtype=torch.float64, device=dev), torch.zeros(d, dtype=torch.float64, device=dev)
    for i in range(0, m, m // 20):
        part = x[i:i + m // 20].double() * s[i:i + m // 20].double() * rstd[i:i + m // 20, None].double()
        total += part.sum(0)
        size += part.abs().sum(0)
    assert bool(((dw.double() - total).abs() <= 2.0**-24 * (m + 4) * size).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [5, 128, 1003, 5120])
def test_eps_is_float32(dev, dtype, d):
    """Rows of zeros, whose rstd is eps's alone, and rows whose mean square is of its size. 1e-5 as float32 lies 2.5e-8 below
    itself, which moves the first row's rstd by a step."""
    mx = _mx()
    x = (_acts(65, d, torch.float32, d, 0.0) * 3e-3).to(dtype)
    x[0] = 0.0
    moved = 0
    for eps in (1e-5, 1e-6, 3e-5):
        y, rstd = mx.rms_norm(x.to(dev), None, eps, return_rstd=True)
        want, _, ref = ob.rms_norm(x, None, eps)
        assert float(rstd[0]) == float(torch.tensor(eps, dtype=torch.float32).double().rsqrt().float())
        assert torch.equal(rstd.cpu(), ref) and torch.equal(y.cpu(), want.to(dtype))
        q, s = mx.rms_norm_quantize_mxfp4(x.to(dev), None, eps)
        check_codes4(q, s, want)
        moved += int((rstd.cpu() != (1.0 / (x.double().square().mean(1) + eps).sqrt()).float()).sum())
    assert moved > 0


def test_weight_of_another_shape_is_refused(dev):
    """Under the name of the function's own norm."""
    mx = _mx()
    x, stat, w = torch.zeros(4, 64, device=dev), torch.ones(4, device=dev), torch.ones(63, device=dev)
    for call in (lambda: mx.rms_norm(x, w), lambda: mx.rms_norm_quantize_fp8(x, w), lambda: mx.rms_norm_quantize_mxfp4(x, w),
                 lambda: mx.rms_norm_backward(x, x, stat, w)):
        with pytest.raises(ValueError, match=r"^rms norm weight of shape \(63,\), expected \(64,\)"):
            call()
    for call in (lambda: mx.layer_norm(x, w), lambda: mx.layer_norm_backward(x, x, stat, stat, w)):
        with pytest.raises(ValueError, match="^layer norm weight of shape"):
            call()


@pytest.mark.parametrize("keep", [False, True])
def test_module_gives_the_gradients_asked_for(dev, keep):
    """Every choice of input, residual and weight; the sum's output alone; no rows."""
    mx = _mx()
    m, d = 19, 264
    x0, r0, dy, ds = (_acts(m, d, torch.bfloat16, i) for i in range(4))
    norm = mx.RMSNorm(d, keep_fp8=keep, device=dev, dtype=torch.bfloat16)
    got = {}
    for choice in range(1, 8):
        x, r = x0.to(dev).requires_grad_(bool(choice & 1)), r0.to(dev).requires_grad_(bool(choice & 2))
        norm.weight.requires_grad_(bool(choice & 4)).grad = None
        y, s = norm(x, r)
        torch.autograd.backward([y, s], [dy.to(dev), ds.to(dev)]) if choice & 3 else y.backward(dy.to(dev))
        for name, t, on in (("x", x, choice & 1), ("r", r, choice & 2), ("w", norm.weight, choice & 4)):
            assert (t.grad is None) == (not on)
            if on:
                assert torch.equal(got.setdefault(name, t.grad.clone()), t.grad)
    assert torch.equal(got["x"], got["r"])
    x, r = x0.to(dev).requires_grad_(), r0.to(dev).requires_grad_()
    norm.weight.grad = None
    norm(x, r)[1].backward(ds.to(dev))
    assert torch.equal(x.grad.cpu(), ds) and torch.equal(r.grad.cpu(), ds) and (norm.weight.grad is None or bool((norm.weight.grad == 0).all()))
    x = x0[:0].to(dev).requires_grad_()
    norm.weight.grad = None
    norm(x).sum().backward()
    assert x.grad.shape == (0, d) and bool((norm.weight.grad == 0).all())
