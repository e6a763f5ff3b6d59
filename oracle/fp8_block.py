"""Block-128 e4m3 format, products, gradients and layer norm in float64 (torch, CPU), from their definitions.

No counterpart in the reference: parity unpinned, the definition is this module's own. A block's exponent e is the
smallest one >= -117 with absmax <= 448 * 2^e over its finite elements (0 for a block of zeros); a value is
rne_e4m3(x / 2^e) * 2^e; NaN and infinities are NaN.
"""

from __future__ import annotations

import torch

BLOCK = 128


def e4m3_table() -> torch.Tensor:
    """The value of each of the 256 codes (sign, 4 exponent bits of bias 7, 3 significand bits; 0x7F and 0xFF NaN)."""
    out = []
    for c in range(256):
        s, e, m = c >> 7, (c >> 3) & 15, c & 7
        v = float("nan") if c & 0x7F == 0x7F else (m / 8 * 2.0**-6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7))
        out.append(-v if s else v)
    return torch.tensor(out, dtype=torch.float64)


def round_e4m3(v: torch.Tensor) -> torch.Tensor:
    """float64 of magnitude <= 448 to the nearest e4m3 value, ties to the even code."""
    _, e = torch.frexp(v.abs().clamp_min(2.0**-6))  # v = m 2^e, m in [0.5, 1): the last place is 2^(e - 4)
    step = torch.ldexp(torch.ones_like(v), e - 4)
    return torch.round(v / step) * step


def exponent(absmax: torch.Tensor) -> torch.Tensor:
    m, e = torch.frexp(absmax)
    e = torch.where(m > 0.875, e - 8, e - 9).clamp_min(-117)
    return torch.where(absmax == 0, torch.zeros_like(e), e)


def _finite_abs(x):
    return torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x))


def rows(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """x [M, K] -> (values float64 [M, K], exponents int [M, ceil(K / 128)])."""
    x = x.double()
    m, k = x.shape
    kb = -(-k // BLOCK)
    xp = torch.zeros(m, kb * BLOCK, dtype=torch.float64)
    xp[:, :k] = x
    e = exponent(_finite_abs(xp).view(m, kb, BLOCK).amax(-1))
    s = torch.ldexp(torch.ones((), dtype=torch.float64), e).repeat_interleave(BLOCK, 1)[:, :k]
    v = round_e4m3(torch.where(torch.isfinite(x), x, torch.zeros_like(x)) / s) * s
    return torch.where(torch.isfinite(x), v, torch.full_like(v, float("nan"))), e


def tiles(w: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """w [N, K] -> (values float64 [N, K], exponents int [ceil(N / 128), ceil(K / 128)])."""
    w = w.double()
    n, k = w.shape
    nb, kb = -(-n // BLOCK), -(-k // BLOCK)
    wp = torch.zeros(nb * BLOCK, kb * BLOCK, dtype=torch.float64)
    wp[:n, :k] = w
    e = exponent(_finite_abs(wp).view(nb, BLOCK, kb, BLOCK).amax((1, 3)))
    s = torch.ldexp(torch.ones((), dtype=torch.float64), e)
    s = s.repeat_interleave(BLOCK, 0).repeat_interleave(BLOCK, 1)[:n, :k]
    v = round_e4m3(torch.where(torch.isfinite(w), w, torch.zeros_like(w)) / s) * s
    return torch.where(torch.isfinite(w), v, torch.full_like(v, float("nan"))), e


def values(q: torch.Tensor, scale: torch.Tensor, block_rows: int = 1) -> torch.Tensor:
    """float64 values of a (codes, scale bytes) pair."""
    v = e4m3_table()[q.cpu().contiguous().view(torch.uint8).long()]
    s = torch.ldexp(torch.ones((), dtype=torch.float64), scale.cpu().contiguous().view(torch.uint8).int() - 127)
    s = s.repeat_interleave(BLOCK, 1)[:, : q.shape[1]].repeat_interleave(block_rows, 0)[: q.shape[0]]
    return v * s


def layer_norm(x, weight, bias, eps):
    """(y, mean, rstd) in float64."""
    x = x.double()
    mean = x.mean(1)
    rstd = 1.0 / (x.var(1, unbiased=False) + eps).sqrt()
    y = (x - mean[:, None]) * rstd[:, None]
    if weight is not None:
        y = y * weight.double()
    return (y if bias is None else y + bias.double()), mean, rstd


def layer_norm_backward(dy, x, mean, rstd, weight):
    """(dx, dweight, dbias) in float64 from the formulas."""
    dy, x, mean, rstd = dy.double(), x.double(), mean.double()[:, None], rstd.double()[:, None]
    xh = (x - mean) * rstd
    g = dy if weight is None else dy * weight.double()
    dx = rstd * (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True))
    return dx, (dy * xh).sum(0), dy.sum(0)
