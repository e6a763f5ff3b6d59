"""Gradients of the 8-bit floating point layer and the layer norm, and the modules that run them, against the formulas in
float64 (oracle/fp8_block.py) and against differences.

Bounds. dW: products of a bfloat16 and an e4m3 value are exact in float32, gradients of float16 and float32 are two and
three such parts, so only float32 additions round: 2^-24 per addend, (parts M + 66) of them (66: the joined slices) on
sum|dy x|. db likewise. dx: the product's bounds (test_gpu_fp8.py). Layer norm: a row's sums are at most 24 additions in
a lane, 6 across lanes and 16 across waves, so 64 * 2^-24 of the sum of magnitudes with room for the few operations
behind; 96 * 2^-24 where two such sums meet.
"""

from __future__ import annotations

import copy

import pytest
import torch

from oracle import fp8_block as ob
from test_gpu_fp8 import DTYPES, _acts, _gen, _half_step, _mx, check_product

pytestmark = pytest.mark.gpu

E = 2.0**-24


def _check_sum(got, ref, magnitude, addends, u=0.0):
    got = got.double().cpu()
    assert got.shape == ref.shape
    bound = E * addends * magnitude + u * ref.abs() * (1 + 2.0**-10) + 1e-300
    err = (got - ref).abs()
    assert bool((err <= bound).all()), f"worst {float((err / bound).max())} of the bound"


BACKWARD = [(1, 1, 1), (1, 16, 128), (3, 17, 129), (31, 64, 256), (33, 130, 100), (64, 300, 205), (129, 256, 512), (257, 515, 260),
            (600, 96, 1000), (2100, 520, 300), (9000, 260, 130)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k", BACKWARD)
def test_linear_backward(dev, dtype, m, n, k):
    mx = _mx()
    x, w = _acts(m, k, dtype, m + 3 * k), _acts(n, k, torch.float32, n + k) * 0.05
    dy = _acts(m, n, dtype, 7 * m + n) * 0.01
    p = mx.prepare_fp8_weight(w.to(dev))
    q, s = mx.quantize_fp8_block128(x.to(dev))
    dx, dw, db = mx.fp8_linear_backward(dy.to(dev), q, s, p)
    xv, wv, gv, d = ob.rows(x)[0], ob.tiles(w)[0], ob.rows(dy)[0], dy.double()
    assert dx.dtype == dtype and dw.dtype == torch.float32 and db.dtype == torch.float32
    check_product(dx, gv, wv.t(), None, m <= 16 or dtype == torch.float32)
    parts = {torch.bfloat16: 1, torch.float16: 2, torch.float32: 3}[dtype]
    _check_sum(dw, d.t() @ xv, d.abs().t() @ xv.abs(), parts * m + 66)
    _check_sum(db, d.sum(0), d.abs().sum(0), m + 66)
    # a contiguous pair, and one gradient at a time: the same bits
    again = mx.fp8_linear_backward(dy.to(dev), q.contiguous(), s.contiguous(), p)
    for a, b in zip(again, (dx, dw, db)):
        assert torch.equal(a, b)
    for i, want in enumerate((dx, dw, db)):
        needs = tuple(j == i for j in range(3))
        got = mx.fp8_linear_backward(dy.to(dev), q, s, p, needs)
        assert torch.equal(got[i], want) and all(got[j] is None for j in range(3) if j != i)


@pytest.mark.parametrize("grad", DTYPES)
def test_gradient_types_and_strides(dev, grad):
    mx = _mx()
    x, w = _acts(150, 333, torch.bfloat16, 1), _acts(272, 333, torch.float32, 2) * 0.05
    wide = _acts(150, 500, torch.bfloat16, 3) * 0.01
    p = mx.prepare_fp8_weight(w.to(dev))
    q, s = mx.quantize_fp8_block128(x.to(dev))
    xv = ob.rows(x)[0]
    for first in (0, 8, 5, 228):  # aligned rows, odd starts, and the last columns of the storage
        dy = wide[:, first : first + 272]
        dx, dw, db = mx.fp8_linear_backward(wide.to(dev)[:, first : first + 272], q, s, p, grad_dtype=grad)
        d = dy.double()
        assert dw.dtype == grad and db.dtype == grad
        u = _half_step(grad) if grad != torch.float32 else 0.0
        _check_sum(dw, d.t() @ xv, d.abs().t() @ xv.abs(), 216, u)
        _check_sum(db, d.sum(0), d.abs().sum(0), 216, u)
        check_product(dx, ob.rows(dy)[0], ob.tiles(w)[0].t(), None, False)
    y3 = mx.fp8_linear_backward(wide.to(dev)[:, :272].reshape(3, 50, 272), q.reshape(3, 50, 333), s.reshape(3, 50, 3), p)
    y2 = mx.fp8_linear_backward(wide.to(dev)[:, :272], q, s, p)
    assert y3[0].shape == (3, 50, 333) and torch.equal(y3[0].reshape(150, 333), y2[0])
    assert torch.equal(y3[1], y2[1]) and torch.equal(y3[2], y2[2])


def test_backward_of_no_rows(dev):
    mx = _mx()
    p = mx.prepare_fp8_weight(torch.randn(40, 256, device=dev))
    q, s = mx.quantize_fp8_block128(torch.zeros(0, 256, device=dev))
    dx, dw, db = mx.fp8_linear_backward(torch.zeros(0, 40, device=dev), q, s, p)
    assert dx.shape == (0, 256)
    assert dw.shape == (40, 256) and not bool(dw.any()) and not bool(db.any())


def test_nan_and_infinities_in_the_gradient(dev):
    """They reach the gradients that read them, and no others."""
    mx = _mx()
    x, w = _acts(100, 256, torch.bfloat16, 1), _acts(160, 256, torch.float32, 2) * 0.05
    p = mx.prepare_fp8_weight(w.to(dev))
    q, s = mx.quantize_fp8_block128(x.to(dev))
    for dtype in DTYPES:
        dy = _acts(100, 160, dtype, 3)
        dy[7, 11], dy[50, 100] = float("nan"), float("inf")
        dx, dw, db = (t.cpu() for t in mx.fp8_linear_backward(dy.to(dev), q, s, p))
        rows = torch.zeros(100, dtype=torch.bool)
        rows[[7, 50]] = True
        assert torch.equal(~torch.isfinite(dx).all(1), rows)
        cols = torch.zeros(160, dtype=torch.bool)
        cols[[11, 100]] = True
        assert torch.equal(~torch.isfinite(dw).all(1), cols) and torch.equal(~torch.isfinite(db), cols)
        assert bool(dw[11].isnan().all()) and bool(db[11].isnan()) and db[100] == float("inf")
        nz = ob.rows(x)[0][50] != 0
        assert bool((dw[100][nz].isinf()).all())


def test_the_same_backward_twice_and_captured(dev):
    """No atomics: the same bits on every run, on two streams and from a replayed graph."""
    mx = _mx()
    x, w = _acts(700, 640, torch.float16, 1), _acts(400, 640, torch.float32, 2) * 0.05
    p = mx.prepare_fp8_weight(w.to(dev))
    q, s = mx.quantize_fp8_block128(x.to(dev))
    dy = (_acts(700, 400, torch.float16, 3) * 0.1).to(dev)
    nx, nw = _acts(700, 640, torch.float16, 4).to(dev), _acts(1, 640, torch.float16, 5)[0].to(dev)

    def step(dy):
        a = mx.fp8_linear_backward(dy, q, s, p)
        y, mean, rstd = mx.layer_norm(nx, nw, None, 1e-6, return_stats=True)
        return (*a, y, *mx.layer_norm_backward(a[0], nx, mean, rstd, nw))

    want = step(dy)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        other = step(dy)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(other, want))
    static = dy.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(static)
    for f in (1.0, -3.0, 0.5):
        static.copy_(dy * f)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, step(static)))


# ---------------------------------------------------------------------------------------
# layer norm
# ---------------------------------------------------------------------------------------

NORMS = [(1, 1), (3, 7), (5, 64), (9, 512), (6, 513), (130, 1000), (4, 1024), (7, 1025), (33, 2048), (5, 4096), (3, 5120), (3, 5376),
         (2, 8192), (3, 8193), (2, 16384), (2, 20480), (2, 24576), (1200, 136)]


def _norm_inputs(m, d, dtype, seed):
    g = _gen(seed)
    x = (torch.randn(m, d, generator=g) * torch.exp(torch.randn(m, 1, generator=g)) + 3 * torch.randn(m, 1, generator=g)).to(dtype)
    w = (1 + 0.3 * torch.randn(d, generator=g)).to(dtype)
    b = (0.3 * torch.randn(d, generator=g)).to(dtype)
    dy = (torch.randn(m, d, generator=g) * 0.1).to(dtype)
    return x, w, b, dy


def _check_norm(y, mean, rstd, x, w, b, eps):
    ry, rm, rr = ob.layer_norm(x, w, b, eps)
    x = x.double()
    near = x.abs().mean(1)
    assert bool(((mean.double().cpu() - rm).abs() <= 64 * E * near + 1e-300).all())
    # the mean's error e enters the variance as e^2
    rel = 64 * E + (64 * E * near * rr) ** 2
    assert bool(((rstd.double().cpu() - rr).abs() <= rel * rr).all())
    wa = torch.ones(x.shape[1], dtype=torch.float64) if w is None else w.double().abs()
    ba = torch.zeros(x.shape[1], dtype=torch.float64) if b is None else b.double().abs()
    xh = (x - rm[:, None]).abs() * rr[:, None]
    bound = _half_step(y.dtype) * ry.abs() + 64 * E * (wa * (near * rr)[:, None] + 2 * wa * xh + ba) + torch.finfo(y.dtype).tiny
    err = (y.double().cpu() - ry).abs()
    assert bool((err <= bound * (1 + 2.0**-7)).all()), float((err / bound).max())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,d", NORMS)
def test_layer_norm(dev, dtype, m, d):
    mx = _mx()
    x, w, b, _ = _norm_inputs(m, d, dtype, m + d)
    y, mean, rstd = mx.layer_norm(x.to(dev), w.to(dev), b.to(dev), 1e-6, return_stats=True)
    assert y.dtype == dtype and mean.dtype == rstd.dtype == torch.float32
    _check_norm(y, mean, rstd, x, w, b, 1e-6)
    assert torch.equal(mx.layer_norm(x.to(dev), w.to(dev), b.to(dev), 1e-6), y)


def _check_norm_grad(got, dy, xv, mean, rstd, w):
    dx, dw, db = got
    rx, rw, rb = ob.layer_norm_backward(dy, xv, mean, rstd, w)
    m, d = xv.shape
    dyd, xd = dy.double(), xv.double()
    xh = ((xd - mean.double()[:, None]) * rstd.double()[:, None]).abs()
    g = (dyd if w is None else dyd * w.double()).abs()
    r = rstd.double()[:, None]
    bound = _half_step(dx.dtype) * rx.abs() + 96 * E * r * (g + g.mean(1, keepdim=True) + xh * (g * xh).mean(1, keepdim=True))
    err = (dx.double().cpu() - rx).abs()
    assert bool((err <= bound * (1 + 2.0**-7) + torch.finfo(dx.dtype).tiny).all()), float((err / bound).max())
    _check_sum(dw, rw, (dyd.abs() * xh).sum(0), m + 70)
    _check_sum(db, rb, dyd.abs().sum(0), m + 70)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,d", NORMS)
def test_layer_norm_backward(dev, dtype, m, d):
    mx = _mx()
    x, w, _, dy = _norm_inputs(m, d, dtype, 5 * m + d)
    _, mean, rstd = ob.layer_norm(x, None, None, 1e-6)
    mean, rstd = mean.float(), rstd.float()
    args = (mean.to(dev), rstd.to(dev), w.to(dev))
    got = mx.layer_norm_backward(dy.to(dev), x.to(dev), *args)
    assert got[0].dtype == dtype and got[1].dtype == got[2].dtype == torch.float32
    _check_norm_grad(got, dy, x, mean, rstd, w)
    # from the input as kept in 8 bits
    pair = mx.quantize_fp8_block128(x.to(dev))
    _check_norm_grad(mx.layer_norm_backward(dy.to(dev), pair, *args), dy, ob.rows(x)[0], mean, rstd, w)
    only = mx.layer_norm_backward(dy.to(dev), x.to(dev), *args, needs_params=False)
    assert torch.equal(only[0], got[0]) and only[1] is None and only[2] is None


@pytest.mark.parametrize("dtype", DTYPES)
def test_layer_norm_parameters_and_strides(dev, dtype):
    mx = _mx()
    x, w, b, dy = _norm_inputs(60, 650, dtype, 1)
    big, gbig = x.to(dev), dy.to(dev)
    for sl in (slice(0, 648), slice(3, 203), slice(8, 136)):
        xv, dv, wv, bv = x[:, sl], dy[:, sl], w[sl], b[sl]
        for pw, pb in ((None, None), (wv, None), (None, bv), (wv.float(), bv.float()), (wv.float(), bv)):
            dw_, db_ = (None if t is None else t.to(dev) for t in (pw, pb))
            y, mean, rstd = mx.layer_norm(big[:, sl], dw_, db_, 1e-5, return_stats=True)
            _check_norm(y, mean, rstd, xv, pw, pb, 1e-5)
            got = mx.layer_norm_backward(gbig[:, sl], big[:, sl], mean, rstd, dw_)
            _check_norm_grad(got, dv, xv, mean.cpu(), rstd.cpu(), pw)
    y3, m3, r3 = mx.layer_norm(big.view(3, 20, 650), w.to(dev), b.to(dev), return_stats=True)
    assert y3.shape == (3, 20, 650) and m3.shape == r3.shape == (3, 20)
    assert torch.equal(y3.view(60, 650), mx.layer_norm(big, w.to(dev), b.to(dev)))
    assert torch.equal(mx.layer_norm_backward(gbig.view(3, 20, 650), big.view(3, 20, 650), m3, r3, w.to(dev))[0].view(60, 650),
                       mx.layer_norm_backward(gbig, big, m3, r3, w.to(dev))[0])
    e = mx.layer_norm(big[:0], w.to(dev))
    assert e.shape == (0, 650)
    z = mx.layer_norm_backward(gbig[:0], big[:0], m3.reshape(-1)[:0], r3.reshape(-1)[:0], w.to(dev))
    assert z[0].shape == (0, 650) and not bool(z[1].any()) and not bool(z[2].any())


def test_layer_norm_of_constant_and_far_rows(dev):
    """Rows without variance, rows far from zero (a variance from squares would cancel), NaN and infinities in one row."""
    mx = _mx()
    x = torch.randn(6, 1000, generator=_gen(1))
    x[1] = 5.0
    x[2] += 1000.0
    x[3, 4] = float("nan")
    x[4, 5] = float("inf")
    y, mean, rstd = mx.layer_norm(x.to(dev), None, None, 1e-6, return_stats=True)
    keep = [0, 1, 2, 5]
    _check_norm(y[keep], mean[keep], rstd[keep], x[keep], None, None, 1e-6)
    assert not bool(y[1].any())
    assert bool(y[3].isnan().all()) and bool(y[4].isnan().all()) and bool(torch.isfinite(y[keep]).all())


def test_gradients_against_differences(dev):
    """<gradient, v> against the difference of the loss along v: the layer's values are linear in each operand, so a whole
    step; the norm's in float64 with a small one."""
    mx = _mx()
    g = _gen(9)

    def grid(*shape):  # values that e4m3 holds at scale 1 (largest 448 in every block, which fixes the scale)
        v = torch.randint(-8, 9, shape, generator=g).float()
        v[..., ::128] = 448.0
        return v

    x, w, dy = grid(96, 256), grid(128, 256), grid(96, 128)
    p = mx.prepare_fp8_weight(w.to(dev))
    q, s = mx.quantize_fp8_block128(x.to(dev))
    dx, dw, db = (t.double().cpu() for t in mx.fp8_linear_backward(dy.to(dev), q, s, p))

    def loss(x, w, b):
        return (dy.double() * (x.double() @ w.double().t() + b.double())).sum()

    zero = torch.zeros(128)
    for grad, at in ((dx, 0), (dw, 1), (db, 2)):
        v = torch.randn(grad.shape, generator=g).double()
        args = [x, w, zero]
        up = list(args)
        up[at] = args[at].double() + v
        diff = loss(*up) - loss(*args)
        assert abs(float((grad * v).sum() - diff)) <= 2.0**-20 * float((grad * v).abs().sum() + loss(*args).abs())
    nx, nw, nb, ndy = (t.double() for t in _norm_inputs(7, 300, torch.float32, 3))
    y, mean, rstd = mx.layer_norm(nx.float().to(dev), nw.float().to(dev), nb.float().to(dev), 1e-5, return_stats=True)
    grads = mx.layer_norm_backward(ndy.float().to(dev), nx.float().to(dev), mean, rstd, nw.float().to(dev))

    def nloss(x, w, b):
        return (ndy * ob.layer_norm(x, w, b, 1e-5)[0]).sum()

    for at, grad in enumerate(grads):
        v = torch.randn(grad.shape, generator=g).double()
        h = 1e-4
        up, down = [nx, nw, nb], [nx, nw, nb]
        up[at], down[at] = up[at] + h * v, down[at] - h * v
        diff = float((nloss(*up) - nloss(*down)) / (2 * h))
        # float32 gradients (2^-20 of the terms) and the difference's own h^2 term
        assert abs(float((grad.double().cpu() * v).sum()) - diff) <= 2.0**-20 * float((grad.double().cpu() * v).abs().sum()) + 1e-5


# ---------------------------------------------------------------------------------------
# modules
# ---------------------------------------------------------------------------------------

@pytest.mark.parametrize("keep", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_norm_and_layer_trained_together(dev, dtype, keep):
    """norm -> layer -> loss through autograd is the composition of the functions, bit for bit, with the input kept in 8 bits."""
    mx = _mx()
    torch.manual_seed(0)
    norm = mx.LayerNorm(328, keep_fp8=keep, device=dev, dtype=dtype)
    layer = mx.Fp8Linear(328, 200, device=dev, dtype=dtype)
    with torch.no_grad():
        norm.weight.uniform_(0.5, 1.5)
        layer.bias.normal_()
    x = _acts(3 * 50, 328, dtype, 1).view(3, 50, 328).to(dev).requires_grad_()
    dy = (_acts(3 * 50, 200, dtype, 2) * 0.1).view(3, 50, 200).to(dev)
    out = layer(norm(x))
    out.backward(dy)
    with torch.no_grad():
        h, mean, rstd = mx.layer_norm(x, norm.weight, norm.bias, norm.eps, return_stats=True)
        p = mx.prepare_fp8_weight(layer.weight)
        assert torch.equal(out, mx.fp8_linear(h, p, layer.bias))
        q, s = mx.quantize_fp8_block128(h)
        dh, dw, db = mx.fp8_linear_backward(dy, q, s, p, grad_dtype=dtype)
        kept = mx.quantize_fp8_block128(x) if keep else x.detach()
        dx, dnw, dnb = mx.layer_norm_backward(dh, kept, mean, rstd, norm.weight)
    assert torch.equal(x.grad, dx) and torch.equal(layer.weight.grad, dw) and torch.equal(layer.bias.grad, db)
    assert torch.equal(norm.weight.grad, dnw.to(dtype)) and torch.equal(norm.bias.grad, dnb.to(dtype))
    # a second backward of a second forward adds up
    layer(norm(x)).backward(dy)
    assert torch.equal(layer.weight.grad, dw + dw)
    # without gradients: the prepared form, the same values
    with torch.no_grad():
        assert torch.equal(layer(norm(x)), out)
        layer.weight.mul_(2.0)
        changed = layer(norm(x))  # (the form follows the parameter)
        assert not torch.equal(changed, out)
        layer.prepare()
        assert torch.equal(layer(norm(x)), changed)


def test_frozen_layer_gives_the_inputs_gradient_only(dev):
    mx = _mx()
    layer = mx.Fp8Linear(256, 96, bias=False, device=dev, dtype=torch.bfloat16)
    layer.weight.requires_grad_(False)
    x = _acts(70, 256, torch.bfloat16, 1).to(dev).requires_grad_()
    y = layer(x)
    assert layer._prepared is not None
    y.sum().backward()
    p = mx.prepare_fp8_weight(layer.weight)
    q, s = mx.quantize_fp8_block128(x.detach())
    assert torch.equal(x.grad, mx.fp8_linear_backward(torch.ones_like(y), q, s, p, (True, False, False))[0])
    assert layer.weight.grad is None


def test_modules_are_not_captured(dev):
    mx = _mx()
    layer, norm = mx.Fp8Linear(128, 64, device=dev, dtype=torch.bfloat16), mx.LayerNorm(128, device=dev, dtype=torch.bfloat16)
    x = torch.randn(4, 128, device=dev, dtype=torch.bfloat16)
    layer.prepare()
    torch.cuda.synchronize()
    for module in (layer, norm):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            with pytest.raises(RuntimeError, match="not captured"):
                module(x)
            with torch.no_grad():
                y = module(x)
        graph.replay()
        torch.cuda.synchronize()
        with torch.no_grad():
            assert torch.equal(y, module(x))


def test_views_that_end_their_storage(dev):
    """Operands that are the last columns of wider tensors: nothing behind their last row is read (the guard values would
    show in no result; the reads' bounds are the kernel's), and the results are those of copies."""
    mx = _mx()
    m, n, k = 150, 272, 384
    x, w = _acts(m, 2 * k, torch.bfloat16, 1), _acts(n, k, torch.float32, 2) * 0.05
    p = mx.prepare_fp8_weight(w.to(dev))
    q, s = mx.quantize_fp8_block128(x.to(dev))
    dy = (_acts(m, 2 * n, torch.bfloat16, 3) * 0.01).to(dev)
    dv, qv, sv = dy[:, n:], q[:, k:], s[:, 3:]
    got = mx.fp8_linear_backward(dv, qv, sv, p)
    want = mx.fp8_linear_backward(dv.contiguous(), qv.contiguous(), sv.contiguous(), p)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert torch.equal(mx.fp8_linear_prequantized(qv, sv, p), mx.fp8_linear_prequantized(qv.contiguous(), sv.contiguous(), p))
    xv, d = ob.rows(x[:, k:])[0], dv.double().cpu()
    _check_sum(got[1], d.t() @ xv, d.abs().t() @ xv.abs(), 216)
    # rows further apart than the products take: copied
    far = torch.zeros(2, 5_000_000, dtype=torch.float8_e4m3fn, device=dev)
    far[:, :k] = q[:2, :k]
    y = mx.fp8_linear_prequantized(far[:, :k], s[:2, :3], p)
    assert torch.equal(y, mx.fp8_linear_prequantized(q[:2, :k].contiguous(), s[:2, :3].contiguous(), p))
    # a gradient that is one value, expanded
    ones = torch.ones((), dtype=torch.bfloat16, device=dev).expand(m, n)
    a, b = mx.fp8_linear_backward(ones, qv, sv, p), mx.fp8_linear_backward(ones.contiguous(), qv, sv, p)
    assert all(torch.equal(u, v) for u, v in zip(a, b))


def test_layer_norm_of_more_rows_than_a_grid_axis(dev):
    """2^26 rows and some: a row per wave is more than 2^32 threads."""
    mx = _mx()
    m = 2**26 + 5
    x = torch.zeros(m, 2, dtype=torch.bfloat16, device=dev)
    x[:, 0] = 1.0
    x[-3:, 1] = 3.0
    y = mx.layer_norm(x, eps=0.0)
    assert bool((y[: m - 3, 0] == 1).all()) and bool((y[: m - 3, 1] == -1).all())
    assert bool((y[m - 3 :, 0] == -1).all()) and bool((y[m - 3 :, 1] == 1).all())


def test_quantizers_from_a_replayed_graph(dev):
    """Each replay gives what an eager call on the same input gives, with eager work between."""
    mx = _mx()
    inputs = [_acts(70, 333, torch.float16, i).to(dev) for i in range(4)]
    w = _acts(200, 333, torch.float32, 9).to(dev)
    static = inputs[0].clone()

    def step(x):
        q, s = mx.quantize_fp8_block128(x)
        p = mx.prepare_fp8_weight(w)
        return (q.view(torch.uint8), s.view(torch.uint8), mx.dequantize_fp8_block128(q, s, torch.float32),
                mx.fp8_linear_prequantized(q, s, p), mx.fp8_linear(x[:9], p), *mx.fp8_linear_backward(mx.fp8_linear(x, p), q, s, p))

    step(static)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(static)
    for x in (inputs[1], inputs[2], inputs[3], inputs[1]):
        static.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        want = step(x)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_the_module_follows_its_weight(dev):
    """Without gradients the layer reads the parameter's present contents: after a step, a load, a move to another type, and
    in a graph that was captured before any eager call."""
    mx = _mx()
    g = _gen(5)
    x = torch.randn(40, 256, generator=g).to(torch.bfloat16).to(dev)
    layer = mx.Fp8Linear(256, 96, device=dev, dtype=torch.float32)

    def fresh():
        return mx.fp8_linear(x, mx.prepare_fp8_weight(layer.weight.detach()), layer.bias.detach())

    graph = torch.cuda.CUDAGraph()
    with torch.no_grad():
        mx.fp8_linear(x, mx.prepare_fp8_weight(layer.weight), layer.bias)
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            captured = layer(x)
        assert torch.equal(layer(x), fresh())
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(captured, fresh())
    before = fresh()
    opt = torch.optim.SGD(layer.parameters(), lr=0.5)
    layer(x).float().sum().backward()
    opt.step()
    with torch.no_grad():
        assert torch.equal(layer(x), fresh()) and not torch.equal(fresh(), before)
        layer.load_state_dict({k: v * 2 for k, v in layer.state_dict().items()})
        assert torch.equal(layer(x), fresh())
        layer.bfloat16()
        assert torch.equal(layer(x), fresh())
        assert layer._form() is layer._form()
        layer.weight = torch.nn.Parameter(layer.weight.detach() * 3)
        assert torch.equal(layer(x), fresh())
        assert torch.equal(copy.deepcopy(layer)(x), fresh())
    layer.weight.requires_grad_(False)
    xg = x.clone().requires_grad_()
    layer(xg).float().sum().backward()
    q, s = mx.quantize_fp8_block128(x)
    want = mx.fp8_linear_backward(torch.ones(40, 96, device=dev, dtype=torch.bfloat16), q, s, mx.prepare_fp8_weight(layer.weight))
    assert torch.equal(xg.grad, want[0])


def test_first_calls_on_two_streams(dev):
    """The layer's hidden form is ordered by the layer: a call on one stream, right behind the call on another that builds
    the form (held back there), reads the built one; and again behind a change of the weight. Its memory is not given out
    while the second stream still reads it."""
    mx = _mx()
    x = _acts(64, 1024, torch.bfloat16, 1).to(dev)
    layer = mx.Fp8Linear(1024, 2048, device=dev, dtype=torch.bfloat16).requires_grad_(False)
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(3):
        want = mx.fp8_linear(x, mx.prepare_fp8_weight(layer.weight), layer.bias)
        torch.cuda.synchronize()
        with torch.cuda.stream(a):
            torch.cuda._sleep(20_000_000)
            ya = layer(x)
        with torch.cuda.stream(b):
            yb = layer(x)
        torch.cuda.synchronize()
        assert torch.equal(ya, want) and torch.equal(yb, want)
        with torch.cuda.stream(b):
            torch.cuda._sleep(20_000_000)
            yb = layer(x)
        with torch.cuda.stream(a):  # (the form's own stream drops it and fills what it gave back)
            other = layer.weight.clone()
            layer.prepare()
            fill = [torch.full_like(t, 127, dtype=torch.uint8) for t in (layer._prepared.q, layer._prepared.qt)]
        torch.cuda.synchronize()
        assert torch.equal(yb, want) and torch.equal(other, layer.weight) and len(fill) == 2
        layer.weight.mul_(-1.5)
        torch.cuda.synchronize()


@pytest.mark.parametrize("eager_first", [False, True])
@pytest.mark.parametrize("frozen", [False, True])
def test_replays_of_the_module_follow_its_weight(dev, eager_first, frozen):
    """Without ``prepare``, a graph's replays read the weight as it is, whether or not an eager call came before."""
    mx = _mx()
    x = _acts(40, 512, torch.bfloat16, 1).to(dev)
    layer = mx.Fp8Linear(512, 384, device=dev, dtype=torch.bfloat16).requires_grad_(not frozen)
    graph = torch.cuda.CUDAGraph()

    def fresh():
        return mx.fp8_linear(x, mx.prepare_fp8_weight(layer.weight), layer.bias)

    with torch.no_grad():
        fresh()
        if eager_first:
            layer(x)
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            y = layer(x)
        for i in range(4):
            graph.replay()
            assert torch.equal(y, fresh())
            layer.weight.mul_(-1.25)
            if i % 2:
                assert torch.equal(layer(x), fresh())


@pytest.mark.parametrize("frozen", [False, True])
def test_replays_read_the_prepared_form_where_it_is(dev, frozen):
    """After ``prepare`` a graph reads the layer's form: a changed weight reaches its replays with the next eager call or
    ``prepare``, in the same memory, whatever else was allocated meanwhile."""
    mx = _mx()
    x = _acts(40, 512, torch.bfloat16, 1).to(dev)
    layer = mx.Fp8Linear(512, 384, device=dev, dtype=torch.bfloat16).requires_grad_(not frozen).prepare()
    graph, others = torch.cuda.CUDAGraph(), []

    def fresh():
        return mx.fp8_linear(x, mx.prepare_fp8_weight(layer.weight), layer.bias)

    with torch.no_grad():
        fresh()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            y = layer(x)
        for i in range(6):
            graph.replay()
            assert torch.equal(y, fresh())
            layer.weight.mul_(-1.25)
            if i % 2:
                layer.prepare()
            else:
                assert torch.equal(layer(x), fresh())
            others += [torch.full_like(t, 127, dtype=torch.uint8) for t in (layer._prepared.q, layer._prepared.qt)]
            torch.cuda.synchronize()


@pytest.mark.parametrize("optimizer", [torch.optim.AdamW, torch.optim.SGD])
def test_evaluation_after_a_fused_step(dev, optimizer):
    """Train, step with a fused optimizer (which does not count its changes), evaluate: the evaluation has the new weight,
    also once the layer is frozen, and in a replayed graph."""
    mx = _mx()
    x = _acts(40, 256, torch.bfloat16, 1).to(dev)
    layer = mx.Fp8Linear(256, 96, device=dev, dtype=torch.float32)
    step, last, graph = optimizer(layer.parameters(), lr=0.05, fused=True), None, torch.cuda.CUDAGraph()
    with torch.no_grad():
        layer(x)
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            captured = layer(x)
    for _ in range(3):
        layer(x).float().square().sum().backward()
        step.step()
        step.zero_grad()
        with torch.no_grad():
            want = mx.fp8_linear(x, mx.prepare_fp8_weight(layer.weight), layer.bias)
            assert torch.equal(layer(x), want) and torch.equal(layer(x), want)
            graph.replay()
            assert torch.equal(captured, want)
        assert last is None or not torch.equal(want, last)
        last = want
        layer.requires_grad_(False)
        assert torch.equal(layer(x), want)
        layer.requires_grad_(True)


def test_inference_loads_and_types_and_back(dev):
    """Contents that change without a count: loaded in inference mode, or rounded by a type and back."""
    mx = _mx()
    x = _acts(40, 256, torch.bfloat16, 1).to(dev)

    def right(layer):
        return torch.equal(layer(x), mx.fp8_linear(x, mx.prepare_fp8_weight(layer.weight), layer.bias))

    with torch.inference_mode():
        layer = mx.Fp8Linear(256, 96, device=dev, dtype=torch.float32).requires_grad_(False)
        for _ in range(3):
            assert right(layer)
            layer.load_state_dict({k: v * -1.5 for k, v in layer.state_dict().items()})
    layer = mx.Fp8Linear(256, 96, device=dev, dtype=torch.float32).requires_grad_(False)
    for _ in range(3):
        layer.weight.add_(0.001)
        assert right(layer)
        layer.bfloat16()
        layer.float()
        assert right(layer)


@pytest.mark.parametrize("wtype,btype", [(torch.bfloat16, torch.float32), (torch.float32, torch.bfloat16), (torch.float16, torch.bfloat16)])
@pytest.mark.parametrize("frozen", [False, True])
def test_parameters_of_two_types(dev, wtype, btype, frozen):
    """Each parameter's gradient is rounded once, to its own type."""
    mx = _mx()
    layer = mx.Fp8Linear(200, 72, device=dev, dtype=wtype)
    layer.bias = torch.nn.Parameter(torch.zeros(72, device=dev, dtype=btype))
    layer.weight.requires_grad_(not frozen)
    x, dy = _acts(90, 200, torch.bfloat16, 1).to(dev), (_acts(90, 72, torch.bfloat16, 2) * 0.1).to(dev)
    layer(x).backward(dy)
    q, s = mx.quantize_fp8_block128(x)
    _, dw, db = mx.fp8_linear_backward(dy, q, s, mx.prepare_fp8_weight(layer.weight), (False, True, True))
    assert layer.bias.grad.dtype == btype and torch.equal(layer.bias.grad, db.to(btype))
    if frozen:
        assert layer.weight.grad is None
    else:
        assert layer.weight.grad.dtype == wtype and torch.equal(layer.weight.grad, dw.to(wtype))


@pytest.mark.parametrize("m", [1, 3])
@pytest.mark.parametrize("far", ["dy", "codes", "scale"])
def test_backward_of_rows_far_apart(dev, far, m):
    """Rows further apart than the weight's gradient reads in place: copied, as the forward pass copies them."""
    mx = _mx()
    n, k = 48, 384
    x, w, dy = _acts(m, k, torch.bfloat16, 1), _acts(n, k, torch.float32, 2) * 0.05, (_acts(m, n, torch.bfloat16, 3) * 0.1).to(dev)
    p = mx.prepare_fp8_weight(w.to(dev))
    q, s = mx.quantize_fp8_block128(x.to(dev))
    want = mx.fp8_linear_backward(dy, q, s, p)

    def apart(t):
        wide = torch.zeros(m, 2**24 + 64, dtype=t.dtype, device=dev)
        wide[:, : t.shape[1]] = t
        return wide[:, : t.shape[1]]

    args = {"dy": dy, "codes": q, "scale": s}
    args[far] = apart(args[far])
    got = mx.fp8_linear_backward(args["dy"], args["codes"], args["scale"], p)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert torch.equal(mx.fp8_linear_prequantized(args["codes"], args["scale"], p), mx.fp8_linear_prequantized(q, s, p))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,n,k", [(7, 64, 200), (33, 130, 100), (600, 96, 1000), (2100, 520, 300)])
def test_full_sums_of_the_inputs_gradient(dev, dtype, m, n, k):
    """dx with every addend; the other gradients are the same bits; and the module passes it on both ways."""
    mx = _mx()
    x, w, dy = _acts(m, k, dtype, 1), _acts(n, k, torch.float32, 2) * 0.05, _acts(m, n, dtype, 3) * 0.01
    p = mx.prepare_fp8_weight(w.to(dev))
    q, s = mx.quantize_fp8_block128(x.to(dev))
    dx, dw, db = mx.fp8_linear_backward(dy.to(dev), q, s, p, full_sums=True)
    check_product(dx, ob.rows(dy)[0], ob.tiles(w)[0].t(), None, True)
    plain = mx.fp8_linear_backward(dy.to(dev), q, s, p)
    assert torch.equal(dw, plain[1]) and torch.equal(db, plain[2])
    layer = mx.Fp8Linear(k, n, bias=False, device=dev, dtype=dtype, full_sums=True)
    with torch.no_grad():
        layer.weight.copy_(w)
    xg = x.to(dev).requires_grad_()
    y = layer(xg)
    y.backward(dy.to(dev))
    p = mx.prepare_fp8_weight(layer.weight)
    assert torch.equal(y, mx.fp8_linear(x.to(dev), p, full_sums=True)) and torch.equal(layer(x.to(dev)), y)
    assert torch.equal(xg.grad, mx.fp8_linear_backward(dy.to(dev), q, s, p, (True, False, False), full_sums=True)[0])
