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
import threading
from dataclasses import dataclass

import torch
from torch.autograd import forward_ad

from . import _lib
from .ops import _OUT_CODES, _bias, _launch, _out_code, _ptr, _raw_stream, _require_gpu, _rows, _vector

BLOCK = 128
_CODES, _SCALE = torch.float8_e4m3fn, torch.float8_e8m0fnu
_MAX_STRIDE = 1 << 22  # of an operand's rows; wider ones are copied
_MAX_GRAD_STRIDE = 1 << 24  # below it, of the rows that the weight's gradient reads


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
    return (torch.empty(m, kb * BLOCK, dtype=_CODES, device=dev),
            torch.empty(m, _ceil(kb, 4), dtype=_SCALE, device=dev))


def _view(t: torch.Tensor, lead: tuple[int, ...], width: int) -> torch.Tensor:
    """The first ``width`` columns of ``t`` as ``[*lead, width]`` (a view)."""
    m, ld = t.shape
    if ld != width:
        t = t.as_strided((m, width), (ld, 1))
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
    """A copy of 1-byte rows with row stride ``ld`` (rounded up to 16), zeros behind them."""
    if t.stride(1) != 1 or (t.shape[0] > 1 and t.stride(0) < t.shape[1]):
        t = t.contiguous()
    m, width = t.shape
    out = torch.empty(m, _ceil(ld, 16), dtype=t.dtype, device=t.device)
    _launch(t.device, "mxq_pad_rows", t.data_ptr(), t.stride(0) if m > 1 else width, width, out.data_ptr(), out.shape[1], m)
    return out


def _operand(q: torch.Tensor, scale: torch.Tensor, k: int):
    """A pair as the matrix products read it: code rows of whole, zero-padded blocks from 16-byte boundaries, scale rows
    of whole words. Pairs of this module's quantizers of whole blocks pass as they are; others are copied."""
    kb = -(-k // BLOCK)
    if k % BLOCK or q.stride(0) % 16 or q.data_ptr() % 16 or not k <= q.stride(0) <= _MAX_STRIDE:
        q = _pad(q, kb * BLOCK)
    if scale.stride(0) % 4 or scale.data_ptr() % 4 or not _ceil(kb, 4) <= scale.stride(0) <= _MAX_STRIDE // 4:
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
    """The values of a ``(codes, scale)`` pair, rounded once to ``out_dtype`` (exact in bf16 and fp32). A value that its code
    rounded past the type's largest is an infinity: float16 inputs from 63488 on, bf16 and fp32 from 1.9375 * 2^127 on."""
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
        code = None
    else:
        code = _float_code(weight, "weight")
    dev = _require_gpu(weight, scale)
    form = PreparedFp8Weight(
        torch.empty(n, kb * BLOCK, dtype=_CODES, device=dev), torch.empty(nb, _ceil(kb, 4), dtype=_SCALE, device=dev),
        torch.empty(k, nb * BLOCK, dtype=_CODES, device=dev) if transposed else None,
        torch.empty(kb, _ceil(nb, 4), dtype=_SCALE, device=dev) if transposed else None, n, k)
    _write_form(form, weight, code, scale)
    return form


def _write_form(form: PreparedFp8Weight, weight: torch.Tensor, code: int | None, scale: torch.Tensor | None = None) -> None:
    """Lays ``weight`` (of dtype ``code``, or codes with ``scale``) out in ``form``'s tensors."""
    n, k = weight.shape
    w = _rows_in_place(weight, k)
    q, s, qt, st = form.q, form.scale, form.qt, form.scale_t
    out = (q.data_ptr(), q.shape[1], s.data_ptr(), s.shape[1], _ptr(qt), 0 if qt is None else qt.shape[1], _ptr(st),
           0 if st is None else st.shape[1], n, k)
    ldw = w.stride(0) if n > 1 else k
    if scale is not None:
        nb, kb = scale.shape
        ws = _rows_in_place(scale, kb)
        _launch(form.device, "mxq_fp8_prepare_tiles", w.data_ptr(), ldw, ws.data_ptr(), ws.stride(0) if nb > 1 else kb, *out)
    else:
        _launch(form.device, "mxq_fp8_quantize_tiles", w.data_ptr(), code, ldw, *out)


# ---------------------------------------------------------------------------------------
# products
# ---------------------------------------------------------------------------------------

@functools.lru_cache(maxsize=4096)
def _workspace(name: str, index: int, *sizes: int) -> int:
    """The library's answer to a workspace query ``name`` for device ``index``, asked with it current."""
    out = ctypes.c_int64()
    with torch.cuda.device(index):
        _lib.call(name, *sizes, ctypes.byref(out))
    return out.value


def _room(need: int, dev) -> torch.Tensor | None:
    return torch.empty(need, dtype=torch.uint8, device=dev) if need else None


def _sums(full: bool) -> int:
    """What an output's type code carries for products that keep every addend."""
    return _lib.FP8_FULL_SUMS if full else 0


def _product(dev, a, sa, m: int, k: int, b, sb, n: int, bias, out_dtype, full_sums: bool) -> torch.Tensor:
    """``[m, n]`` of operands in the products' layout."""
    out = torch.empty(m, n, dtype=out_dtype, device=dev)
    code = _out_code(out_dtype) | _sums(full_sums)
    if m == 0:
        return out
    need = _workspace("mxq_fp8_gemm_workspace", dev.index, m, n, k)
    ws = _room(need, dev)
    _launch(dev, "mxq_fp8_gemm", a.data_ptr(), a.stride(0), sa.data_ptr(), sa.stride(0), b.data_ptr(), b.stride(0), sb.data_ptr(),
            sb.stride(0), _ptr(bias), out.data_ptr(), n, code, m, n, k, _ptr(ws), need)
    return out


def _check_weight(weight: PreparedFp8Weight, k: int) -> None:
    if not isinstance(weight, PreparedFp8Weight):
        raise TypeError(f"weight must come from prepare_fp8_weight, got {type(weight).__name__}")
    if k != weight.in_features:
        raise ValueError(f"K mismatch: {k} vs {weight.in_features}")


def fp8_linear(x: torch.Tensor, weight: PreparedFp8Weight, bias: torch.Tensor | None = None,
               out_dtype: torch.dtype | None = None, full_sums: bool = False) -> torch.Tensor:
    """``x @ weight.T + bias`` with ``x [..., K]`` quantized as :func:`quantize_fp8_block128` does; ``out_dtype`` defaults
    to ``x``'s. Up to 16 rows are quantized inside the product's launch.

    bf16 and fp16 results of more than 16 rows come from an instruction that cuts each of 64 addends below 2^-13 of the
    largest of them: beside those types' own rounding little on a layer's usual data (5e-5 to 2e-4 of the results' root
    mean square), at worst 64 * 2^-13 of the largest for every 64. ``full_sums`` keeps every addend to float32's
    precision, at half the rate; float32 results and up to 16 rows always do.
    """
    if x.dim() < 1 or x.shape[-1] == 0:
        raise ValueError("fp8_linear needs a non-empty last dimension")
    _check_weight(weight, x.shape[-1])
    xcode = _float_code(x, "input")
    dev = _require_gpu(x, weight.q, bias)
    out_dtype = out_dtype or x.dtype
    code = _out_code(out_dtype) | _sums(full_sums)
    n, k = weight.out_features, weight.in_features
    bias = _bias(bias, n, out_dtype, dev)
    x2 = _rows_in_place(x, k)
    m = x2.shape[0]
    out = torch.empty(m, n, dtype=out_dtype, device=dev)
    if m:
        q, s = weight.q, weight.scale
        need = _workspace("mxq_fp8_linear_workspace", dev.index, m, n, k)
        ws = _room(need, dev)
        _launch(dev, "mxq_fp8_linear", x2.data_ptr(), xcode, x2.stride(0) if m > 1 else k, q.data_ptr(), q.shape[1], s.data_ptr(),
                s.shape[1], _ptr(bias), out.data_ptr(), n, code, m, n, k, _ptr(ws), need)
    return out if x.dim() == 2 else out.reshape(*x.shape[:-1], n)


def fp8_linear_prequantized(q: torch.Tensor, scale: torch.Tensor, weight: PreparedFp8Weight, bias: torch.Tensor | None = None,
                            out_dtype: torch.dtype = torch.bfloat16, full_sums: bool = False) -> torch.Tensor:
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
    out = _product(dev, q, scale, m, k, weight.q, weight.scale, n, bias, out_dtype, full_sums)
    return out if len(shape) == 2 else out.reshape(*shape[:-1], n)


# ---------------------------------------------------------------------------------------
# gradients
# ---------------------------------------------------------------------------------------

def _readable(t: torch.Tensor, width: int) -> bool:
    """Whether every row of ``t`` (1-byte elements) can be read ``width`` wide from 16-byte boundaries."""
    m, ld = t.shape[0], t.stride(0)
    if t.data_ptr() % 16 or (m > 1 and (ld % 16 or not width <= ld < _MAX_GRAD_STRIDE)):
        return False
    return t.untyped_storage().nbytes() - t.storage_offset() >= (m - 1) * ld + width


def fp8_linear_backward(dy: torch.Tensor, q: torch.Tensor, scale: torch.Tensor, weight: PreparedFp8Weight,
                        needs: tuple[bool, bool, bool] = (True, True, True), grad_dtype: torch.dtype = torch.float32,
                        full_sums: bool = False):
    """Gradients ``(dx, dweight, dbias)`` of :func:`fp8_linear` from the output's gradient ``dy [..., N]``, the input as it
    was kept in 8 bits (the pair ``q [..., K]``, ``scale``) and the prepared weight; ``needs`` says which (``None`` for the
    others). The quantizers pass gradients through unchanged.

    ``dx = dY^ W^`` in ``dy``'s dtype, ``dY^`` being ``dy`` quantized as an activation is (``full_sums`` as in
    :func:`fp8_linear`); ``dweight = dy^T X^`` and
    ``dbias = sum dy`` in ``grad_dtype``, from ``dy`` itself: with float32 sums of exact products where ``dy`` is bf16,
    fp16 or (to 24 bits) fp32, which go through the matrix instructions as one, two or three bfloat16 parts.
    """
    shape = q.shape
    q, scale, m, k = _pair(q, scale)
    _check_weight(weight, k)
    code = _float_code(dy, "gradient")
    gcode = _out_code(grad_dtype)
    n = weight.out_features
    if tuple(dy.shape) != (*shape[:-1], n):
        raise ValueError(f"gradient of shape {tuple(dy.shape)}, expected {(*shape[:-1], n)}")
    want_x, want_w, want_b = needs
    if want_x and weight.qt is None:
        raise ValueError("the input's gradient needs the transposed weight (prepare_fp8_weight(..., transposed=True))")
    dev = _require_gpu(dy, q, scale, weight.q)
    y = _rows_in_place(dy, n)
    ldy = y.stride(0) if m > 1 else n
    direct = dy.dtype == torch.bfloat16 and n % 16 == 0 and ldy % 8 == 0 and ldy < _MAX_GRAD_STRIDE and y.data_ptr() % 16 == 0
    readable = _readable(q, _ceil(k, 16))
    if m > 1 and scale.stride(0) >= _MAX_GRAD_STRIDE:
        scale = scale.contiguous()
    dx = torch.empty(m, k, dtype=dy.dtype, device=dev) if want_x else None
    dw = torch.empty(n, k, dtype=grad_dtype, device=dev) if want_w else None
    db = torch.empty(n, dtype=grad_dtype, device=dev) if want_b else None
    # (without rows dx is empty, and its pointer may be null)
    needs = (1 if want_x and m else 0) | (2 if want_w else 0) | (4 if want_b else 0)
    if needs:
        need = _workspace("mxq_fp8_linear_backward_workspace", dev.index, m, n, k, code, direct, readable, needs)
        ws = _room(need, dev)
        bt, st = weight.qt, weight.scale_t
        _launch(dev, "mxq_fp8_linear_backward", y.data_ptr(), code | _sums(full_sums), ldy, direct, q.data_ptr(),
                q.stride(0) if m > 1 else _ceil(k, 16) if readable else k, scale.data_ptr(),
                scale.stride(0) if m > 1 else scale.shape[1], readable, _ptr(bt), bt.shape[1] if want_x else 0,
                _ptr(st), st.shape[1] if want_x else 0, dx.data_ptr() if want_x and m else None,
                _ptr(dw), _ptr(db), gcode, m, n, k, _ptr(ws), need)
    if want_x and len(shape) != 2:
        dx = dx.reshape(shape)
    return dx, dw, db


# ---------------------------------------------------------------------------------------
# layer norm
# ---------------------------------------------------------------------------------------

def _norm_params(d: int, dev, dtype, weight, bias, what: str = "layer norm"):
    """Weight and bias as the kernels read them: both of x's dtype or both float32."""
    target = dtype
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None:
            if t.shape != (d,):
                raise ValueError(f"{what} {name} of shape {tuple(t.shape)}, expected ({d},)")
            if t.dtype != dtype:
                target = torch.float32
    return (None if weight is None else _vector(weight, target, dev), None if bias is None else _vector(bias, target, dev),
            _OUT_CODES[target])


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None, eps: float = 1e-5,
               return_stats: bool = False):
    """``(x - mean) * rstd * weight + bias`` over the last dimension (at most 24576), in float32 and rounded once to ``x``'s
    dtype. ``return_stats`` adds the rows' float32 ``mean`` and ``rstd``, which :func:`layer_norm_backward` takes."""
    code = _float_code(x, "input")
    if x.dim() < 1 or x.shape[-1] == 0:
        raise ValueError("layer_norm needs a non-empty last dimension")
    if not eps >= 0:
        raise ValueError(f"eps must not be negative, got {eps}")
    dev = _require_gpu(x, weight, bias)
    d = x.shape[-1]
    w, b, pcode = _norm_params(d, dev, x.dtype, weight, bias)
    x2 = _rows_in_place(x, d)
    m = x2.shape[0]
    y = torch.empty(m, d, dtype=x.dtype, device=dev)
    mean = torch.empty(m, dtype=torch.float32, device=dev) if return_stats else None
    rstd = torch.empty(m, dtype=torch.float32, device=dev) if return_stats else None
    if m:
        _launch(dev, "mxq_layer_norm", x2.data_ptr(), code, x2.stride(0) if m > 1 else max(x2.stride(0), d), _ptr(w), _ptr(b), pcode,
                float(eps), y.data_ptr(), _ptr(mean), _ptr(rstd), m, d)
    y = y if x.dim() == 2 else y.reshape(x.shape)
    if not return_stats:
        return y
    if x.dim() != 2:
        mean, rstd = mean.reshape(x.shape[:-1]), rstd.reshape(x.shape[:-1])
    return y, mean, rstd


def layer_norm_backward(dy: torch.Tensor, x, mean: torch.Tensor, rstd: torch.Tensor, weight: torch.Tensor | None = None,
                        needs_params: bool = True):
    """Gradients ``(dx, dweight, dbias)`` of :func:`layer_norm`: ``dx`` in ``dy``'s dtype, the other two in float32 (``None``
    without ``needs_params``). ``x`` is the forward's input, or that input as it was kept in 8 bits, a ``(codes, scale)``
    pair of :func:`quantize_fp8_block128`; ``mean`` and ``rstd`` are the forward's."""
    code = _float_code(dy, "gradient")
    if dy.dim() < 1 or dy.shape[-1] == 0:
        raise ValueError("layer_norm_backward needs a non-empty last dimension")
    d = dy.shape[-1]
    if isinstance(x, (tuple, list)):
        if tuple(x[0].shape) != tuple(dy.shape):
            raise ValueError(f"input of shape {tuple(x[0].shape)} for a gradient of shape {tuple(dy.shape)}")
        x2, xs, _, _ = _pair(*x)
        xcode, ldxs = _lib.DTYPE_E4M3, max(xs.stride(0), xs.shape[1])
    else:
        if tuple(x.shape) != tuple(dy.shape):
            raise ValueError(f"input of shape {tuple(x.shape)} for a gradient of shape {tuple(dy.shape)}")
        if x.dtype != dy.dtype:
            raise ValueError(f"input of {x.dtype} for a gradient of {dy.dtype}")
        x2, xs, xcode, ldxs = _rows_in_place(x, d), None, code, 0
    y2 = _rows_in_place(dy, d)
    m = y2.shape[0]
    for name, t in (("mean", mean), ("rstd", rstd)):
        if t.dtype != torch.float32 or t.numel() != m:
            raise ValueError(f"{name} must be float32 with one entry per row ({m}), got {t.dtype} {tuple(t.shape)}")
    dev = _require_gpu(dy, x2, xs, mean, rstd, weight)
    w, _, pcode = _norm_params(d, dev, dy.dtype, weight, None)
    dx = torch.empty(m, d, dtype=dy.dtype, device=dev)
    both = torch.empty(2, d, dtype=torch.float32, device=dev) if needs_params else None
    need = _workspace("mxq_layer_norm_backward_workspace", dev.index, m, d) if needs_params else 0
    ws = _room(need, dev)
    if m or needs_params:
        mean, rstd = _vector(mean, torch.float32, dev), _vector(rstd, torch.float32, dev)
        _launch(dev, "mxq_layer_norm_backward", y2.data_ptr(), code, max(y2.stride(0), d), x2.data_ptr(), xcode, max(x2.stride(0), d),
                _ptr(xs), ldxs, mean.data_ptr(), rstd.data_ptr(), _ptr(w), pcode, dx.data_ptr(), _ptr(both), m, d, _ptr(ws), need)
    dx = dx if dy.dim() == 2 else dx.reshape(dy.shape)
    if not needs_params:
        return dx, None, None
    dw, db = both.unbind(0)
    return dx, dw, db


# ---------------------------------------------------------------------------------------
# modules
# ---------------------------------------------------------------------------------------

def _capturing(device: torch.device) -> bool:
    """Whether ``device``'s current stream is being captured into a graph."""
    if device.type != "cuda":
        return False
    if torch.cuda.current_device() == device.index:
        return torch.cuda.is_current_stream_capturing()
    with torch.cuda.device(device):
        return torch.cuda.is_current_stream_capturing()


def _refuse_capture(device: torch.device) -> None:
    """Autograd keeps one accumulation node per parameter, bound to the stream of its first use, for as long as any graph
    holds it: a backward pass captured while an eager graph of the same parameters lives would join that stream and
    end the process. A training step is captured through the functions, which own no such nodes."""
    if _capturing(device):
        raise RuntimeError("the autograd modules are not captured into graphs; capture fp8_linear, fp8_linear_backward, "
                           "mxfp4_linear, mxfp4_linear_backward, layer_norm, layer_norm_backward, rms_norm and "
                           "rms_norm_backward instead")


def _refuse_tangents(*tensors: torch.Tensor | None) -> None:
    """Forward-mode tangents, which the kernels do not carry on (a tensor that has one need not require a gradient)."""
    if getattr(forward_ad, "_current_level", 0) < 0:  # (no level is open: 2 us less of a call's 10)
        return
    for t in tensors:
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise RuntimeError("the autograd modules have no forward mode: their inputs and parameters take no tangents")


class _Fp8LinearFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, prepared, full_sums):
        dev = _require_gpu(x, prepared.q, bias)
        _refuse_capture(dev)
        q, s, m, k = _quantize_rows(x)
        n = prepared.out_features
        y = _product(dev, q, s, m, k, prepared.q, prepared.scale, n, _bias(bias, n, x.dtype, dev), x.dtype, full_sums)
        # the input leaves the graph in 8 bits: only the pair is kept
        ctx.save_for_backward(q, s, prepared.qt, prepared.scale_t)
        ctx.sizes, ctx.full_sums = (x.shape, n, k), full_sums
        ctx.dtypes = (None if weight is None else weight.dtype, None if bias is None else bias.dtype)
        return y.reshape(*x.shape[:-1], n)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        _refuse_capture(dy.device)
        q, s, qt, st = ctx.saved_tensors
        shape, n, k = ctx.sizes
        wdtype, bdtype = ctx.dtypes
        want_x, want_w, want_b = ctx.needs_input_grad[:3]
        weight = PreparedFp8Weight(q, s, qt, st, n, k)  # (the gradients read the transposed copy only)
        m = q.shape[0]
        # of two types (or a float64 bias's alone), in float32, each then rounded once to its own
        wanted = {t for t, want in ((wdtype, want_w), (bdtype, want_b)) if want}
        own = wanted.pop() if len(wanted) == 1 else None
        dx, dw, db = fp8_linear_backward(dy.reshape(m, n), q[:, :k], s[:, : -(-k // BLOCK)], weight, (want_x, want_w, want_b),
                                         own if own in _OUT_CODES else torch.float32, ctx.full_sums)
        return (dx.reshape(shape) if want_x else None, dw.to(wdtype) if want_w else None, db.to(bdtype) if want_b else None,
                None, None)


def _event(device: torch.device):
    """An event behind all that ``device``'s current stream has been given."""
    event = torch.cuda.Event()
    event.record(torch.cuda.current_stream(device))
    return event


def _follow(device: torch.device, event, tensors) -> None:
    """Puts ``device``'s current stream behind ``event`` and holds the memory of ``tensors`` until its work on them is done."""
    stream = torch.cuda.current_stream(device)
    stream.wait_event(event)
    for t in tensors:
        t.record_stream(stream)


def _synchronize(device: torch.device) -> None:
    torch.cuda.synchronize(device)


def _state(weight: torch.Tensor) -> tuple:
    """What changes with a parameter's contents: the parameter, its storage and its count of changes in place."""
    return (weight,), weight.data_ptr(), weight.dtype, weight.device, None if weight.is_inference() else weight._version


class _Kept:
    """A weight's 8-bit form that a layer keeps between calls, and what it was built from (``of``; ``None``: of nothing that
    still holds). The call that builds it writes memory that its caller does not see, so the order of the streams that use
    it is kept here: one other than the builder's waits for the build, and the memory is not given out again while it
    reads. ``asked``: by the layer's user, who has waited for it. A graph reads only such a form, in place (``captured``);
    ``held`` are the forms that graphs read and that no longer fit the weight. ``shared``: another stream, or a backward
    pass to come, reads the form."""

    __slots__ = ("form", "of", "asked", "captured", "shared", "held", "home", "stream", "built")

    def __init__(self, form: PreparedFp8Weight, of: tuple, asked: bool, held: tuple = ()):
        self.form, self.captured, self.shared, self.held = form, False, False, held
        self.home = _raw_stream(form.device.index)  # (the stream whose memory the form is)
        self.done(of, asked)

    def done(self, of: tuple, asked: bool) -> None:
        """The current stream has been given the build."""
        self.of, self.asked = of, asked
        self.stream, self.built = _raw_stream(self.form.device.index), _event(self.form.device)

    def forget(self) -> None:
        self.of, self.asked = None, False

    def holds(self, weight: torch.Tensor) -> bool:
        """Whether ``weight`` is what the form was built from, by all that is counted of it."""
        return self.of is not None and self.of[0][0] is weight and self.of[1:] == _state(weight)[1:]

    def fits(self, weight: torch.Tensor, transposed: bool) -> bool:
        f = self.form
        return (weight.shape == (f.out_features, f.in_features) and weight.device == f.device and
                (f.qt is not None or not transposed))

    def alone(self) -> bool:
        """Whether only earlier work of the current stream reads the form."""
        return not self.shared and self.stream == _raw_stream(self.form.device.index)

    def tensors(self) -> list[torch.Tensor]:
        f = self.form
        return [t for t in (f.q, f.scale, f.qt, f.scale_t) if t is not None]

    def use(self) -> PreparedFp8Weight:
        """The form, for work on the current stream."""
        device = self.form.device
        stream = _raw_stream(device.index)
        if stream != self.stream or stream != self.home:
            self.shared = True
            _follow(device, self.built, self.tensors())
        return self.form


_KEPT_LOCK = threading.RLock()  # (calls of one layer from several threads)


class Fp8Linear(torch.nn.Module):
    """A linear layer computed in 8-bit floating point, for serving and for training.

    ``weight`` ``[out_features, in_features]`` and ``bias`` are ordinary parameters (bf16, fp16 or fp32). A frozen
    weight is read in its 8-bit form, built by :meth:`prepare` or the first call, and again once the parameter was moved,
    loaded or changed in place (changes through ``.data`` are not seen: call :meth:`prepare`). One that needs a gradient, or
    was made in inference mode, has the form built from the parameter in every call, since fused optimizers and inference
    mode change it unseen; without gradients :meth:`prepare` saves that. What the backward pass keeps of the input is its
    8-bit pair (:func:`fp8_linear_backward`). The quantizers pass gradients through unchanged. Activations are bf16, fp16
    or fp32.

    Calls without gradients can be captured into a graph. Its replays build the form from the parameter's contents each
    time, unless :meth:`prepare` was called first: then they read that form. ``full_sums`` as in :func:`fp8_linear`, for
    the layer's results and its input's gradient.
    """

    def __init__(self, in_features: int, out_features: int, bias: bool = True, device=None, dtype=None, full_sums: bool = False):
        super().__init__()
        self.in_features, self.out_features, self.full_sums = in_features, out_features, full_sums
        self.weight = torch.nn.Parameter(torch.empty(out_features, in_features, device=device, dtype=dtype))
        self.bias = torch.nn.Parameter(torch.zeros(out_features, device=device, dtype=dtype)) if bias else None
        torch.nn.init.normal_(self.weight, std=in_features**-0.5)
        self._kept: _Kept | None = None

    @property
    def _prepared(self) -> PreparedFp8Weight | None:
        return None if self._kept is None else self._kept.form

    def __getstate__(self):
        return {**self.__dict__, "_kept": None}  # (copies and pickles build their own)

    def __setstate__(self, state):
        state = {k: v for k, v in state.items() if k not in ("_prepared", "_prepared_of")}
        super().__setstate__({"_kept": None, "full_sums": False, **state})

    def _state(self) -> tuple:
        return _state(self.weight)

    def _forget(self) -> None:
        if self._kept is not None:
            self._kept.forget()

    def _apply(self, fn, recurse: bool = True):
        out = super()._apply(fn, recurse)
        with _KEPT_LOCK:  # (a type and back can return the storage and count of before with rounded contents)
            self._forget()
            if self._kept is not None and not self._kept.captured:
                self._kept = None
        return out

    def _load_from_state_dict(self, *args, **kwargs):
        super()._load_from_state_dict(*args, **kwargs)
        self._forget()

    def train(self, mode: bool = True):
        if self.weight.requires_grad or not (self._kept is not None and self._kept.asked):
            self._forget()
        return super().train(mode)

    def _build(self, asked: bool, transposed: bool) -> _Kept:
        """The kept form anew from the parameter's present contents; in the same memory where a graph reads it, or where
        nothing else can be reading it."""
        weight, kept = self.weight.detach(), self._kept
        with torch.inference_mode(False):  # (tensors made in that mode cannot be saved for a backward pass)
            if kept is None or not kept.fits(weight, transposed) or not (kept.captured or kept.alone()):
                held = () if kept is None else kept.held + ((kept.form,) if kept.captured else ())
                self._kept = _Kept(prepare_fp8_weight(weight, transposed=transposed), self._state(), asked, held)
            else:
                if kept.captured:  # (replays may be under way on any stream, and follow on any)
                    _synchronize(weight.device)
                _write_form(kept.form, weight, _float_code(weight, "weight"))
                torch.autograd.graph.increment_version(kept.tensors())  # (backward passes that saved them refuse to run)
                if kept.captured:
                    _synchronize(weight.device)
                kept.done(self._state(), asked)
        return self._kept

    def prepare(self) -> "Fp8Linear":
        """Builds the weight's 8-bit form from its present contents, for calls without weight gradients, and waits for it.
        The form is taken for the weight's until the parameter is seen to change, moved or loaded, until a forward with
        gradients of the weight, and, unless it is frozen, until :meth:`train` or :meth:`eval`. Calls captured into graphs
        read it where it is: later changes of the weight reach their replays with the next ``prepare`` or eager call."""
        if _capturing(self.weight.device):
            raise RuntimeError("Fp8Linear.prepare is not captured into graphs: call it before the capture")
        with _KEPT_LOCK:
            _synchronize(self._build(True, True).form.device)
        return self

    def _form(self, saved: bool = False) -> PreparedFp8Weight:
        """The form for one call; ``saved``: a backward pass will read it too."""
        weight = self.weight
        with _KEPT_LOCK:
            kept = self._kept
            # Not every change in place is counted: fused optimizers and changes of inference tensors are not. A form of a
            # weight that is open to them is the weight's for one call only, unless it was asked for.
            current = (kept is not None and kept.holds(weight) and (kept.form.qt is not None or not saved) and
                       (kept.asked or not (weight.requires_grad or weight.is_inference())))
            if _capturing(weight.device):
                if current and kept.asked:
                    kept.captured = True
                    return kept.form
                return prepare_fp8_weight(weight, transposed=False)  # (part of the graph: its replays follow the weight)
            if not current:
                kept = self._build(False, saved or not weight.requires_grad)
            form = kept.use()
            kept.shared |= saved
            return form

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if x.dim() < 1 or x.shape[-1] != self.in_features:
            raise ValueError(f"input of shape {tuple(x.shape)} for a layer of {self.in_features} input features")
        weight, bias = self.weight, self.bias
        _refuse_tangents(x, weight, bias)
        if not torch.is_grad_enabled() or not (x.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad)):
            return fp8_linear(x, self._form(), bias, full_sums=self.full_sums)
        if weight.requires_grad:
            self._forget()
            prepared = prepare_fp8_weight(weight)
        else:
            prepared = self._form(saved=True)
        return _Fp8LinearFn.apply(x, weight, bias, prepared, self.full_sums)

    def extra_repr(self) -> str:
        return f"in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}"


class _LayerNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, keep_fp8):
        _refuse_capture(x.device)
        y, mean, rstd = layer_norm(x, weight, bias, eps, return_stats=True)
        kept = quantize_fp8_block128(x) if keep_fp8 else (x,)
        ctx.save_for_backward(mean, rstd, weight, *kept)
        ctx.dtypes = tuple(None if t is None else t.dtype for t in (weight, bias))
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        _refuse_capture(dy.device)
        mean, rstd, weight, *kept = ctx.saved_tensors
        want_x, want_w, want_b = ctx.needs_input_grad[:3]
        x = tuple(kept) if len(kept) == 2 else kept[0]
        dx, dw, db = layer_norm_backward(dy, x, mean, rstd, weight, needs_params=want_w or want_b)
        return (dx if want_x else None, dw.to(ctx.dtypes[0]) if want_w else None, db.to(ctx.dtypes[1]) if want_b else None,
                None, None)


class LayerNorm(torch.nn.Module):
    """Layer norm over the last dimension (:func:`layer_norm`) with a learned weight and bias. ``keep_fp8`` keeps the input
    for the backward pass in 8 bits instead of as it is."""

    def __init__(self, features: int, eps: float = 1e-5, bias: bool = True, keep_fp8: bool = False, device=None, dtype=None):
        super().__init__()
        self.features, self.eps, self.keep_fp8 = features, eps, keep_fp8
        self.weight = torch.nn.Parameter(torch.ones(features, device=device, dtype=dtype))
        self.bias = torch.nn.Parameter(torch.zeros(features, device=device, dtype=dtype)) if bias else None

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if x.dim() < 1 or x.shape[-1] != self.features:
            raise ValueError(f"input of shape {tuple(x.shape)} for a norm of {self.features} features")
        weight, bias = self.weight, self.bias
        _refuse_tangents(x, weight, bias)
        if not torch.is_grad_enabled() or not (x.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad)):
            return layer_norm(x, weight, bias, self.eps)
        return _LayerNormFn.apply(x, weight, bias, self.eps, self.keep_fp8)

    def extra_repr(self) -> str:
        return f"{self.features}, eps={self.eps}, bias={self.bias is not None}, keep_fp8={self.keep_fp8}"
