"""The 8-bit floating point layer: quantizers, product, gradients, and activations kept in 8 bits.

The format is e4m3 codes with a power of two per block of 128: 1 x 128 for activations and gradients, 128 x 128 for
weights, the scales as E8M0 bytes, which gfx950's matrix instructions apply themselves. Block scales are the smallest
2^e (e >= -117) with ``absmax <= 448 * 2^e``; codes are ``x / 2^e`` rounded once to nearest even; NaN and infinities
become NaN in their own place. An activation's ``(codes, scale)`` pair is all that the backward pass needs of it: the
pair that a layer's forward multiplied, or any other tensor put away by :func:`quantize_fp8_block128`.

No counterpart in the reference. Every function runs the HIP kernels of libmx_qlinear.so on the tensors' GPU and
current stream; there is no CPU path.
"""

from __future__ import annotations

import ctypes
import functools
from dataclasses import dataclass

import torch

from . import _lib
from .ops import _OUT_CODES, _bias, _launch, _out_code, _ptr, _require_gpu, _rows

BLOCK = 128
_CODES, _SCALE = torch.float8_e4m3fn, torch.float8_e8m0fnu
# rows up to which a product streams the weight (mxq_fp8_linear_rows), and those it quantizes on the way
_FEW_ROWS, _FUSED_ROWS = 64, 16


def _ceil(n: int, to: int) -> int:
    return -(-n // to) * to


def _float_code(t: torch.Tensor, what: str) -> int:
    code = _OUT_CODES.get(t.dtype)
    if code is None:
        raise ValueError(f"unsupported {what} dtype {t.dtype}")
    return code


def _rows_in_place(x: torch.Tensor, width: int) -> torch.Tensor:
    """``x`` as ``[rows, width]`` with unit column stride, copied only where its layout has no such form."""
    if x.dim() == 2 and x.stride(1) == 1 and x.stride(0) >= width:
        return x
    return _rows(x, width)


def _new_pair(m: int, k: int, dev) -> tuple[torch.Tensor, torch.Tensor]:
    """Storage for codes and scales of [m, k]: rows of whole blocks, scale rows of whole words."""
    kb = -(-k // BLOCK)
    return (torch.empty((m, kb * BLOCK), dtype=_CODES, device=dev),
            torch.empty((m, _ceil(kb, 4)), dtype=_SCALE, device=dev))


def _view(t: torch.Tensor, lead: tuple[int, ...], width: int) -> torch.Tensor:
    """The first ``width`` columns of ``t`` as ``[*lead, width]`` (a view)."""
    if t.shape[1] != width:
        t = t[:, :width]
    return t if len(lead) == 1 else t.unflatten(0, lead) if lead else t.squeeze(0)


def _pair(q: torch.Tensor, scale: torch.Tensor, what: str = "activation"):
    """A ``(codes, scale)`` pair as 2-D tensors with unit column stride: (codes, scale, M, K)."""
    if q.dtype != _CODES or scale.dtype != _SCALE:
        raise ValueError(f"an 8-bit {what} is float8_e4m3fn codes with float8_e8m0fnu scales, got {q.dtype} and "
                         f"{scale.dtype}")
    if q.dim() < 1 or q.shape[-1] == 0:
        raise ValueError(f"an 8-bit {what} needs a non-empty last dimension")
    k = q.shape[-1]
    kb = -(-k // BLOCK)
    if scale.shape != (*q.shape[:-1], kb):
        raise ValueError(f"scale of shape {tuple(scale.shape)} for codes of shape {tuple(q.shape)}: expected "
                         f"{(*q.shape[:-1], kb)}")
    if q.dim() != 2:
        lead = q.shape[:-1].numel()
        q, scale = q.reshape(lead, k), scale.reshape(lead, kb)
    if q.stride(1) != 1 or (q.shape[0] > 1 and q.stride(0) < k):
        q = q.contiguous()
    if scale.stride(1) != 1 or (scale.shape[0] > 1 and scale.stride(0) < kb):
        scale = scale.contiguous()
    return q, scale, q.shape[0], k


def _pad(t: torch.Tensor, ld: int) -> torch.Tensor:
    """A copy of 1-byte rows with row stride ``ld``, zeros behind them."""
    out = torch.zeros((t.shape[0], ld), dtype=torch.uint8, device=t.device)
    out[:, : t.shape[1]] = t.view(torch.uint8)
    return out.view(t.dtype)


def _operand(q: torch.Tensor, scale: torch.Tensor, k: int):
    """A pair as the matrix products read it: code rows of whole, zero-padded blocks from 16-byte boundaries, scale rows
    of whole words. Pairs of this module's quantizers of whole blocks pass as they are; others are copied."""
    kb = -(-k // BLOCK)
    if k % BLOCK or q.stride(0) % 16 or q.data_ptr() % 16 or q.stride(0) < k:
        q = _pad(q, kb * BLOCK)
    if scale.stride(0) % 4 or scale.data_ptr() % 4 or scale.stride(0) < _ceil(kb, 4):
        scale = _pad(scale, _ceil(kb, 4))
    return q, scale


# ---------------------------------------------------------------------------------------
# quantizers
# ---------------------------------------------------------------------------------------

def _quantize_rows(x: torch.Tensor):
    """The quantizer's storage: (codes [M, ceil(K / 128) * 128], scales [M, whole words], M, K)."""
    code = _float_code(x, "input")
    dev = _require_gpu(x)
    if x.dim() < 1 or x.shape[-1] == 0:
        raise ValueError("an 8-bit quantizer needs a non-empty last dimension")
    k = x.shape[-1]
    x2 = _rows_in_place(x, k)
    m = x2.shape[0]
    q, s = _new_pair(m, k, dev)
    if m:
        _launch(dev, "mxq_fp8_quantize_rows", x2.data_ptr(), code, max(x2.stride(0), k), q.data_ptr(), q.shape[1], s.data_ptr(),
                s.shape[1], m, k)
    return q, s, m, k


def quantize_fp8_block128(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """``x [..., K]`` (bf16, fp16 or fp32) in 8 bits: ``(codes float8_e4m3fn [..., K], scale float8_e8m0fnu
    [..., ceil(K / 128)])``, one scale per row and 128 columns; the last block of a row may be short.

    The tensors are views of rows padded to whole blocks (scales: to whole words) where ``K`` is not one.
    """
    q, s, _, k = _quantize_rows(x)
    lead = tuple(x.shape[:-1])
    return _view(q, lead, k), _view(s, lead, -(-k // BLOCK))


def dequantize_fp8_block128(q: torch.Tensor, scale: torch.Tensor, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values of a ``(codes, scale)`` pair, rounded once to ``out_dtype`` (exact in bf16 and fp32)."""
    code = _out_code(out_dtype)
    dev = _require_gpu(q, scale)
    shape = q.shape
    q, scale, m, k = _pair(q, scale)
    out = torch.empty(shape, dtype=out_dtype, device=dev)
    if m:
        _launch(dev, "mxq_fp8_dequantize_rows", q.data_ptr(), max(q.stride(0), k), scale.data_ptr(),
                max(scale.stride(0), scale.shape[1]), out.data_ptr(), code, m, k)
    return out


@dataclass(frozen=True)
class PreparedFp8Weight:
    """An 8-bit weight as the products read it (:func:`prepare_fp8_weight`): codes ``q [N, K rounded up]`` with
    ``scale``, and the transposed copy ``qt [K, N rounded up]`` with ``scale_t`` that the input's gradient
    multiplies by (``None`` without it)."""

    q: torch.Tensor
    scale: torch.Tensor
    qt: torch.Tensor | None
    scale_t: torch.Tensor | None
    out_features: int
    in_features: int

    @property
    def device(self) -> torch.device:
        return self.q.device


def prepare_fp8_weight(weight: torch.Tensor, scale: torch.Tensor | None = None, transposed: bool = True) -> PreparedFp8Weight:
    """A layer's weight ``[N, K]`` for :func:`fp8_linear`: quantized by 128 x 128 tiles (bf16, fp16 or fp32), or, with
    ``scale`` (float8_e8m0fnu ``[ceil(N / 128), ceil(K / 128)]``), codes that are float8_e4m3fn already. ``transposed``
    also lays out the transposed copy, which :func:`fp8_linear_backward` needs for the input's gradient."""
    if weight.dim() != 2 or weight.shape[0] == 0 or weight.shape[1] == 0:
        raise ValueError(f"weight must be a non-empty 2D [out_features, in_features], got {tuple(weight.shape)}")
    weight = weight.detach()
    n, k = weight.shape
    nb, kb = -(-n // BLOCK), -(-k // BLOCK)
    if scale is not None:
        if weight.dtype != _CODES or scale.dtype != _SCALE:
            raise ValueError(f"a quantized weight is float8_e4m3fn codes with float8_e8m0fnu scales, got {weight.dtype} and "
                             f"{scale.dtype}")
        if tuple(scale.shape) != (nb, kb):
            raise ValueError(f"weight scale of shape {tuple(scale.shape)}, expected {(nb, kb)}")
        _require_gpu(weight, scale)
        # (byte copies at load: torch's own)
        qt = _pad(weight.view(torch.uint8).t(), nb * BLOCK).view(_CODES) if transposed else None
        st = _pad(scale.view(torch.uint8).t(), _ceil(nb, 4)).view(_SCALE) if transposed else None
        return PreparedFp8Weight(_pad(weight, kb * BLOCK), _pad(scale, _ceil(kb, 4)), qt, st, n, k)
    code = _float_code(weight, "weight")
    dev = _require_gpu(weight)
    w = _rows_in_place(weight, k)
    q = torch.empty((n, kb * BLOCK), dtype=_CODES, device=dev)
    s = torch.empty((nb, _ceil(kb, 4)), dtype=_SCALE, device=dev)
    qt = torch.empty((k, nb * BLOCK), dtype=_CODES, device=dev) if transposed else None
    st = torch.empty((kb, _ceil(nb, 4)), dtype=_SCALE, device=dev) if transposed else None
    _launch(dev, "mxq_fp8_quantize_tiles", w.data_ptr(), code, w.stride(0), q.data_ptr(), q.shape[1], s.data_ptr(), s.shape[1],
            _ptr(qt), nb * BLOCK, _ptr(st), _ceil(nb, 4), n, k)
    return PreparedFp8Weight(q, s, qt, st, n, k)


# ---------------------------------------------------------------------------------------
# products
# ---------------------------------------------------------------------------------------

@functools.lru_cache(maxsize=4096)
def _gemm_bytes(m: int, n: int, k: int, index: int) -> int:
    out = ctypes.c_int64()
    with torch.cuda.device(index):
        _lib.call("mxq_fp8_gemm_workspace", m, n, k, ctypes.byref(out))
    return out.value


def _product(dev, a, sa, m: int, k: int, b, sb, n: int, bias, out_dtype) -> torch.Tensor:
    """``[m, n]`` of operands in the products' layout."""
    out = torch.empty((m, n), dtype=out_dtype, device=dev)
    code = _out_code(out_dtype)
    if m == 0:
        return out
    if m <= _FEW_ROWS:
        _launch(dev, "mxq_fp8_linear_rows", a.data_ptr(), _lib.DTYPE_E4M3, a.stride(0), sa.data_ptr(), sa.stride(0), b.data_ptr(),
                b.stride(0), sb.data_ptr(), sb.stride(0), _ptr(bias), out.data_ptr(), n, code, m, n, k)
        return out
    need = _gemm_bytes(m, n, k, dev.index)
    ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    _launch(dev, "mxq_fp8_gemm", a.data_ptr(), a.stride(0), sa.data_ptr(), sa.stride(0), b.data_ptr(), b.stride(0), sb.data_ptr(),
            sb.stride(0), _ptr(bias), out.data_ptr(), n, code, m, n, k, _ptr(ws), need)
    return out


def _check_weight(weight: PreparedFp8Weight, k: int) -> None:
    if not isinstance(weight, PreparedFp8Weight):
        raise TypeError(f"weight must come from prepare_fp8_weight, got {type(weight).__name__}")
    if k != weight.in_features:
        raise ValueError(f"K mismatch: {k} vs {weight.in_features}")


def fp8_linear(x: torch.Tensor, weight: PreparedFp8Weight, bias: torch.Tensor | None = None,
               out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """``x @ weight.T + bias`` with ``x [..., K]`` quantized as :func:`quantize_fp8_block128` does; ``out_dtype`` defaults
    to ``x``'s. Up to 16 rows are quantized inside the product's launch."""
    if x.dim() < 1 or x.shape[-1] == 0:
        raise ValueError("fp8_linear needs a non-empty last dimension")
    _check_weight(weight, x.shape[-1])
    xcode = _float_code(x, "input")
    dev = _require_gpu(x, weight.q, bias)
    out_dtype = out_dtype or x.dtype
    code = _out_code(out_dtype)
    n, k = weight.out_features, weight.in_features
    bias = _bias(bias, n, out_dtype, dev)
    m = x.numel() // k
    if 0 < m <= _FUSED_ROWS and k % 8 == 0:
        x2 = _rows_in_place(x, k)
        ld = x2.stride(0) if m > 1 else k
        if x2.data_ptr() % 16 == 0 and ld * x2.element_size() % 16 == 0:
            out = torch.empty((m, n), dtype=out_dtype, device=dev)
            _launch(dev, "mxq_fp8_linear_rows", x2.data_ptr(), xcode, ld, None, 0, weight.q.data_ptr(), weight.q.shape[1],
                    weight.scale.data_ptr(), weight.scale.shape[1], _ptr(bias), out.data_ptr(), n, code, m, n, k)
            return out if x.dim() == 2 else out.reshape(*x.shape[:-1], n)
    q, s, m, k = _quantize_rows(x)
    out = _product(dev, q, s, m, k, weight.q, weight.scale, n, bias, out_dtype)
    return out if x.dim() == 2 else out.reshape(*x.shape[:-1], n)


def fp8_linear_prequantized(q: torch.Tensor, scale: torch.Tensor, weight: PreparedFp8Weight, bias: torch.Tensor | None = None,
                            out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """:func:`fp8_linear` of an input that is a ``(codes, scale)`` pair already."""
    shape = q.shape
    q, scale, m, k = _pair(q, scale)
    _check_weight(weight, k)
    dev = _require_gpu(q, scale, weight.q, bias)
    _out_code(out_dtype)
    n = weight.out_features
    bias = _bias(bias, n, out_dtype, dev)
    if m:
        q, scale = _operand(q, scale, k)
    out = _product(dev, q, scale, m, k, weight.q, weight.scale, n, bias, out_dtype)
    return out if len(shape) == 2 else out.reshape(*shape[:-1], n)
