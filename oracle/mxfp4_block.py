"""MXFP4 format, products, the input's gradient, and the rms norm in float64 (torch, CPU), from their definitions.

No counterpart in the reference: parity unpinned, the definition is this module's own. A block is 32 columns of a row; its
exponent e is the smallest one >= -125 with absmax <= 6 * 2^e (0 for a block of zeros), a value rne_e2m1(x / 2^e) * 2^e; a
block with a NaN or an infinity is NaN throughout (scale byte 255).
"""

from __future__ import annotations

import torch

BLOCK = 32
VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def table() -> torch.Tensor:
    """The value of each of the 16 codes (bit 3 the sign)."""
    return torch.tensor([*VALUES, *(-v for v in VALUES)], dtype=torch.float64)


def round_e2m1(v: torch.Tensor) -> torch.Tensor:
    """Codes of float64 of magnitude <= 6, to the nearest value, ties to the even code: by the distances to all eight."""
    grid = torch.tensor(VALUES, dtype=torch.float64)
    d = (v.abs().unsqueeze(-1) - grid).abs()
    near = d == d.amin(-1, keepdim=True)
    even = near & (torch.arange(8) % 2 == 0)
    pick = torch.where(even.any(-1, keepdim=True), even, near)
    code = pick.to(torch.uint8).argmax(-1)
    return (code + torch.where(torch.signbit(v), 8, 0)).to(torch.uint8)


def exponent(absmax: torch.Tensor) -> torch.Tensor:
    m, e = torch.frexp(absmax)
    e = torch.where(m > 0.75, e - 2, e - 3).clamp_min(-125)
    return torch.where(absmax == 0, torch.zeros_like(e), e)


def rows(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """x [M, K] -> (values float64 [M, K], scale bytes int [M, ceil(K / 32)], codes uint8 [M, K])."""
    x = x.double()
    m, k = x.shape
    kb = -(-k // BLOCK)
    xp = torch.zeros(m, kb * BLOCK, dtype=torch.float64)
    xp[:, :k] = x
    xb = xp.view(m, kb, BLOCK)
    bad = ~torch.isfinite(xb).all(-1)
    xb = torch.where(bad[..., None], torch.zeros_like(xb), xb)
    e = exponent(xb.abs().amax(-1))
    s = torch.ldexp(torch.ones((), dtype=torch.float64), e)
    codes = round_e2m1(xb / s[..., None])
    codes = torch.where(bad[..., None], torch.zeros_like(codes), codes)
    v = table()[codes.long()] * s[..., None]
    v = torch.where(bad[..., None], torch.full_like(v, float("nan")), v)
    return v.view(m, -1)[:, :k], torch.where(bad, 255, e + 127).int(), codes.view(m, -1)[:, :k]


def pack(codes: torch.Tensor) -> torch.Tensor:
    """Codes uint8 [M, K] two per byte, the even column's in the low four bits."""
    m, k = codes.shape
    c = torch.zeros(m, -(-k // 2) * 2, dtype=torch.uint8)
    c[:, :k] = codes
    return c[:, 0::2] | (c[:, 1::2] << 4)


def unpack(q: torch.Tensor, k: int) -> torch.Tensor:
    q = q.cpu().contiguous().view(torch.uint8)
    return torch.stack((q & 15, q >> 4), -1).view(q.shape[0], -1)[:, :k]


def values(q: torch.Tensor, scale: torch.Tensor, k: int) -> torch.Tensor:
    """float64 values of a (codes, scale bytes) pair of k columns."""
    b = scale.cpu().contiguous().view(torch.uint8).int()
    s = torch.ldexp(torch.ones((), dtype=torch.float64), b - 127)
    s = torch.where(b == 255, torch.full_like(s, float("nan")), s)
    return table()[unpack(q, k).long()] * s.repeat_interleave(BLOCK, 1)[:, :k]


def tiles(scale: torch.Tensor, k: int) -> dict[int, int]:
    """Where each scale byte of [rows, ceil(k / 32)] lies in the products' tiles: {offset: byte}."""
    groups = -(-k // 512)
    out = {}
    for r in range(scale.shape[0]):
        for b in range(scale.shape[1]):
            c = b % 16
            out[(r // 32 * groups + b // 16) * 512 + (c // 4) % 2 * 256 + r % 32 * 8 + c // 8 * 4 + c % 4] = int(scale[r, b])
    return out


def rms_norm(x, weight, eps, residual=None):
    """(y float32, s in x's dtype, rstd float32) with the roundings of the definition: s to x's dtype, eps to float32, rstd once
    from float64, s * rstd and the product with the weight to float32."""
    s = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    eps = float(torch.tensor(eps, dtype=torch.float32))
    rstd = (1.0 / (s.double().square().mean(1) + eps).sqrt()).float()
    return normed(s, rstd, weight), s, rstd


def normed(s, rstd, weight):
    y = s.float() * rstd[:, None]
    return y if weight is None else y * weight.float()


def rms_norm_backward(dy, s, rstd, weight, dsum=None):
    """(dx, dweight) in float64 from the formulas."""
    dy, s, r = dy.double(), s.double(), rstd.double()[:, None]
    xh = s * r
    g = dy if weight is None else dy * weight.double()
    dx = r * (g - xh * (g * xh).mean(1, keepdim=True))
    return dx if dsum is None else dx + dsum.double(), (dy * xh).sum(0)
