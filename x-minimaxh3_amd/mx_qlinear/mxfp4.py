"""The microscaled 4-bit layer (MXFP4): quantizer, product, the input's gradient through a frozen weight.

The format is e2m1 codes (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives), two in a byte, the even column's in the low four
bits, with a power of two (an E8M0 byte) per 1 x 32 block of a row, for activations and weights alike: what gfx950's 4-bit
matrix instructions read. Block scales are the smallest 2^e (e >= -125) with ``absmax <= 6 * 2^e``, so no value is cut off;
codes are ``x / 2^e`` rounded once to nearest even. e2m1 has no NaN: a block with a NaN or an infinity has the scale byte
255 and is NaN throughout. Pairs of other making are taken too: any code and scale byte (the input's gradient may count weights
below 2^-126, which only the bytes 0 and 1 make, as zeros, and takes one that is past float32's range, 2^128 and more, as an
infinity, with fp16 and fp32 gradients also as NaN; the quantizer makes one of an element from 3.5 * 2^126 on).

No counterpart in the reference. Every function runs the HIP kernels of libmx_qlinear.so on the tensors' GPU and current
stream; there is no CPU path.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

from .fp8 import _ceil, _float_code, _refuse_capture, _refuse_tangents, _room, _rows_in_place, _view, _workspace
from .ops import _OUT_CODES, _bias, _launch, _out_code, _ptr, _require_gpu

BLOCK = 32
_CODES, _SCALE = torch.float4_e2m1fn_x2, torch.float8_e8m0fnu
_MAX_STRIDE = 1 << 22  # bytes, of rows of codes that the product reads in place
_MAX_GRAD_STRIDE = 1 << 24  # below it, of the rows that the input's gradient reads in place


def _row_bytes(k: int) -> int:
    """Bytes of a weight's row of codes as the products read it."""
    return _ceil(k, 512) // 2


def _scale_bytes(rows: int, k: int) -> int:
    """Bytes of the scale tiles of [rows, k]."""
    return -(-rows // 32) * -(-k // 512) * 512


def _pair(q: torch.Tensor, scale: torch.Tensor, width: int | None, what: str = "activation"):
    """A ``(codes, scale)`` pair as 2-D tensors of one-byte elements with unit column stride: (codes, scale, M, K)."""
    if q.dtype != _CODES or scale.dtype != _SCALE:
        raise ValueError(f"a 4-bit {what} is float4_e2m1fn_x2 codes with float8_e8m0fnu scales, got {q.dtype} and {scale.dtype}")
    if q.dim() < 1 or q.shape[-1] == 0:
        raise ValueError(f"a 4-bit {what} needs a non-empty last dimension")
    half = q.shape[-1]
    k = 2 * half if width is None else width
    if -(-k // 2) != half:
        raise ValueError(f"codes of shape {tuple(q.shape)} (two in an element) for a width of {k}")
    kb = -(-k // BLOCK)
    if scale.shape != (*q.shape[:-1], kb):
        raise ValueError(f"scale of shape {tuple(scale.shape)} for codes of shape {tuple(q.shape)}: expected "
                         f"{(*q.shape[:-1], kb)}")
    if q.dim() != 2:
        lead = q.shape[:-1].numel()
        q, scale = q.view(torch.uint8).reshape(lead, half), scale.reshape(lead, kb)
    m, (ldq, one), (lds, each) = q.shape[0], q.stride(), scale.stride()
    if one != 1 or (m > 1 and ldq < half):
        q = q.view(torch.uint8).contiguous()
    if each != 1 or (m > 1 and lds < kb):
        scale = scale.contiguous()
    return q, scale, m, k


# ---------------------------------------------------------------------------------------
# quantizer
# ---------------------------------------------------------------------------------------

def _new_pair(m: int, k: int, dev) -> tuple[torch.Tensor, torch.Tensor]:
    """Storage for codes and scales of [m, k]: rows of whole 128 columns."""
    n = -(-k // 128)
    if torch.are_deterministic_algorithms_enabled():  # (it then fills what it allocates, which it cannot in the codes' type)
        q = torch.empty(m, n * 64, dtype=torch.uint8, device=dev).view(_CODES)
    else:
        q = torch.empty(m, n * 64, dtype=_CODES, device=dev)
    return q, torch.empty(m, n * 4, dtype=_SCALE, device=dev)


def _as_pair(q: torch.Tensor, s: torch.Tensor, lead: tuple[int, ...], k: int) -> tuple[torch.Tensor, torch.Tensor]:
    return _view(q, lead, -(-k // 2)), _view(s, lead, -(-k // BLOCK))


def quantize_mxfp4(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """``x [..., K]`` (bf16, fp16 or fp32) in 4 bits: ``(codes float4_e2m1fn_x2 [..., ceil(K / 2)], scale float8_e8m0fnu
    [..., ceil(K / 32)])``, one scale per row and 32 columns; the last block of a row may be short, and the last code of an
    odd row stands alone in its byte.

    The tensors are views of rows padded to whole 128 columns where ``K`` is not.
    """
    code = _float_code(x, "input")
    dev = _require_gpu(x)
    if x.dim() < 1 or x.shape[-1] == 0:
        raise ValueError("a 4-bit quantizer needs a non-empty last dimension")
    k = x.shape[-1]
    x2 = _rows_in_place(x, k)
    m = x2.shape[0]
    q, s = _new_pair(m, k, dev)
    if m:
        _launch(dev, "mxq_mxfp4_quantize_rows", x2.data_ptr(), code, max(x2.stride(0), k), q.data_ptr(), q.shape[1], s.data_ptr(),
                s.shape[1], m, k)
    return _as_pair(q, s, tuple(x.shape[:-1]), k)


def dequantize_mxfp4(q: torch.Tensor, scale: torch.Tensor, out_dtype: torch.dtype = torch.bfloat16,
                     width: int | None = None) -> torch.Tensor:
    """The values of a ``(codes, scale)`` pair, rounded once to ``out_dtype`` (exact in bf16 and fp32). ``width`` is the
    number of columns, twice the codes' elements unless given: an odd one leaves the last byte's high code out. A value that
    its code rounded past the type's largest is an infinity."""
    code = _out_code(out_dtype)
    dev = _require_gpu(q, scale)
    lead = q.shape[:-1]
    q, scale, m, k = _pair(q, scale, width)
    out = torch.empty(*lead, k, dtype=out_dtype, device=dev)
    if m:
        _launch(dev, "mxq_mxfp4_dequantize_rows", q.data_ptr(), max(q.stride(0), q.shape[1]), scale.data_ptr(),
                max(scale.stride(0), scale.shape[1]), out.data_ptr(), code, m, k)
    return out


# ---------------------------------------------------------------------------------------
# weights
# ---------------------------------------------------------------------------------------

@dataclass(frozen=True)
class PreparedMxfp4Weight:
    """A 4-bit weight as the products read it (:func:`prepare_mxfp4_weight`): code rows ``q`` uint8 ``[N, bytes]`` of whole 256
    bytes and ``scale`` uint8 in tiles of 32 rows x 16 blocks."""

    q: torch.Tensor
    scale: torch.Tensor
    out_features: int
    in_features: int

    @property
    def device(self) -> torch.device:
        return self.q.device


def prepare_mxfp4_weight(weight: torch.Tensor, scale: torch.Tensor | None = None, in_features: int | None = None) -> PreparedMxfp4Weight:
    """A layer's weight ``[N, K]`` for :func:`mxfp4_linear`: quantized by 1 x 32 blocks (bf16, fp16 or fp32), or, with ``scale``
    (float8_e8m0fnu ``[N, ceil(K / 32)]``), float4_e2m1fn_x2 codes ``[N, ceil(K / 2)]`` that are there already, of
    ``in_features`` columns (twice the codes' elements unless given)."""
    if weight.dim() != 2 or weight.shape[0] == 0 or weight.shape[1] == 0:
        raise ValueError(f"weight must be a non-empty 2D [out_features, in_features], got {tuple(weight.shape)}")
    weight = weight.detach()
    n = weight.shape[0]
    if scale is None:
        code = _float_code(weight, "weight")
        if in_features is not None and in_features != weight.shape[1]:
            raise ValueError(f"in_features={in_features} for a weight of shape {tuple(weight.shape)}")
        k = weight.shape[1]
    else:
        q, s, _, k = _pair(weight, scale, in_features, "weight")
    dev = _require_gpu(weight, scale)
    with torch.inference_mode(False):  # (tensors made in that mode cannot be saved for a backward pass)
        out = torch.empty(n, _row_bytes(k), dtype=torch.uint8, device=dev)
        # (the places of a last tile's missing rows, which no product uses: the same bytes for the same weight)
        tiles = (torch.empty if n % 32 == 0 else torch.zeros)(_scale_bytes(n, k), dtype=torch.uint8, device=dev)
    if scale is None:
        w = _rows_in_place(weight, k)
        _launch(dev, "mxq_mxfp4_quantize_rows", w.data_ptr(), code, w.stride(0) if n > 1 else k, out.data_ptr(), out.shape[1],
                tiles.data_ptr(), 0, n, k)
    else:
        _launch(dev, "mxq_mxfp4_layout", q.data_ptr(), q.stride(0) if n > 1 else q.shape[1], s.data_ptr(),
                s.stride(0) if n > 1 else s.shape[1], out.data_ptr(), out.shape[1], tiles.data_ptr(), n, k)
    return PreparedMxfp4Weight(out, tiles, n, k)


def _check_weight(weight: PreparedMxfp4Weight, k: int) -> None:
    if not isinstance(weight, PreparedMxfp4Weight):
        raise TypeError(f"weight must come from prepare_mxfp4_weight, got {type(weight).__name__}")
    if k != weight.in_features:
        raise ValueError(f"K mismatch: {k} vs {weight.in_features}")


# ---------------------------------------------------------------------------------------
# products
# ---------------------------------------------------------------------------------------

def mxfp4_linear(x: torch.Tensor, weight: PreparedMxfp4Weight, bias: torch.Tensor | None = None,
                 out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """``x @ weight.T + bias`` with ``x [..., K]`` quantized as :func:`quantize_mxfp4` does; ``out_dtype`` defaults to ``x``'s.
    Up to 16 rows, or fewer of a long ``K``, are quantized inside the product's launch. Sums are float32: a block's 32
    products are added exactly, and the blocks' sums with what lies below 2^-22 of the largest cut."""
    if x.dim() < 1 or x.shape[-1] == 0:
        raise ValueError("mxfp4_linear needs a non-empty last dimension")
    _check_weight(weight, x.shape[-1])
    xcode = _float_code(x, "input")
    dev = _require_gpu(x, weight.q, bias)
    out_dtype = out_dtype or x.dtype
    code = _out_code(out_dtype)
    n, k = weight.out_features, weight.in_features
    bias = _bias(bias, n, out_dtype, dev)
    x2 = _rows_in_place(x, k)
    m = x2.shape[0]
    out = torch.empty(m, n, dtype=out_dtype, device=dev)
    if m:
        q = weight.q
        need = _workspace("mxq_mxfp4_linear_workspace", dev.index, m, n, k)
        ws = _room(need, dev)
        _launch(dev, "mxq_mxfp4_linear", x2.data_ptr(), xcode, x2.stride(0) if m > 1 else k, q.data_ptr(), q.shape[1],
                weight.scale.data_ptr(), _ptr(bias), out.data_ptr(), n, code, m, n, k, _ptr(ws), need)
    return out if x.dim() == 2 else out.reshape(*x.shape[:-1], n)


def mxfp4_linear_prequantized(q: torch.Tensor, scale: torch.Tensor, weight: PreparedMxfp4Weight, bias: torch.Tensor | None = None,
                              out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """:func:`mxfp4_linear` of an input that is a ``(codes, scale)`` pair already; up to 16 rows, or fewer of a long
    ``K``, are one launch."""
    if not isinstance(weight, PreparedMxfp4Weight):
        raise TypeError(f"weight must come from prepare_mxfp4_weight, got {type(weight).__name__}")
    lead = q.shape[:-1]
    q, scale, m, k = _pair(q, scale, weight.in_features)
    dev = _require_gpu(q, scale, weight.q, bias)
    code = _out_code(out_dtype)
    n = weight.out_features
    bias = _bias(bias, n, out_dtype, dev)
    out = torch.empty(m, n, dtype=out_dtype, device=dev)
    if m:
        ldq = q.stride(0) if m > 1 else q.shape[1]
        direct = k % 256 == 0 and ldq % 16 == 0 and ldq <= _MAX_STRIDE and q.data_ptr() % 16 == 0
        need = _workspace("mxq_mxfp4_linear_prequantized_workspace", dev.index, m, n, k, direct)
        ws = _room(need, dev)
        _launch(dev, "mxq_mxfp4_linear_prequantized", q.data_ptr(), ldq, scale.data_ptr(), scale.stride(0) if m > 1 else scale.shape[1],
                direct, weight.q.data_ptr(), weight.q.shape[1], weight.scale.data_ptr(), _ptr(bias), out.data_ptr(), n, code, m, n, k,
                _ptr(ws), need)
    return out if len(lead) == 1 else out.reshape(*lead, n)


def mxfp4_linear_backward(dy: torch.Tensor, weight: PreparedMxfp4Weight, needs: tuple[bool, bool] = (True, True),
                          grad_dtype: torch.dtype = torch.float32):
    """Gradients ``(dx, dbias)`` of :func:`mxfp4_linear` through a frozen weight, from the output's gradient ``dy [..., N]``;
    ``needs`` says which (``None`` for the other). The quantizer passes gradients through unchanged.

    ``dx = dy W^`` in ``dy``'s dtype and ``dbias = sum dy`` in ``grad_dtype``, from ``dy`` as it is: float32 sums of products
    that are exact where ``dy`` is bf16, fp16 or (to 24 bits, from 2^-103 up) fp32, which go through the matrix instructions as
    one, two or three bfloat16 parts; an fp32 value that bfloat16 rounds to an infinity, ``(2 - 2^-8) 2^127`` and more, is one.
    """
    if not isinstance(weight, PreparedMxfp4Weight):
        raise TypeError(f"weight must come from prepare_mxfp4_weight, got {type(weight).__name__}")
    code = _float_code(dy, "gradient")
    gcode = _out_code(grad_dtype)
    n, k = weight.out_features, weight.in_features
    if dy.dim() < 1 or dy.shape[-1] != n:
        raise ValueError(f"gradient of shape {tuple(dy.shape)} for a layer of {n} output features")
    want_x, want_b = needs
    dev = _require_gpu(dy, weight.q)
    y = _rows_in_place(dy, n)
    m = y.shape[0]
    ldy = y.stride(0) if m > 1 else n
    direct = (dy.dtype == torch.bfloat16 and n % 8 == 0 and ldy % 8 == 0 and ldy < _MAX_GRAD_STRIDE and y.data_ptr() % 16 == 0)
    dx = torch.empty(m, k, dtype=dy.dtype, device=dev) if want_x else None
    db = torch.empty(n, dtype=grad_dtype, device=dev) if want_b else None
    # (without rows dx is empty, and its pointer may be null)
    wants = (1 if want_x and m else 0) | (2 if want_b else 0)
    if wants:
        need = _workspace("mxq_mxfp4_linear_backward_workspace", dev.index, m, n, k, code, direct, wants)
        ws = _room(need, dev)
        _launch(dev, "mxq_mxfp4_linear_backward", y.data_ptr(), code, ldy, direct, weight.q.data_ptr(), weight.q.shape[1],
                weight.scale.data_ptr(), dx.data_ptr() if want_x and m else None, _ptr(db), gcode, m, n, k, _ptr(ws), need)
    if want_x and dy.dim() != 2:
        dx = dx.reshape(*dy.shape[:-1], k)
    return dx, db


# ---------------------------------------------------------------------------------------
# module
# ---------------------------------------------------------------------------------------

class _Mxfp4LinearFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, qweight, scale, bias, sizes):
        _refuse_capture(x.device)
        ctx.save_for_backward(qweight, scale)
        ctx.sizes, ctx.bias_dtype = sizes, None if bias is None else bias.dtype
        return mxfp4_linear(x, PreparedMxfp4Weight(qweight, scale, *sizes), bias)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        _refuse_capture(dy.device)
        qweight, scale = ctx.saved_tensors
        want_x, want_b = ctx.needs_input_grad[0], ctx.needs_input_grad[3]
        # (a float64 bias's gradient is summed in float32)
        dx, db = mxfp4_linear_backward(dy, PreparedMxfp4Weight(qweight, scale, *ctx.sizes), (want_x, want_b),
                                       ctx.bias_dtype if ctx.bias_dtype in _OUT_CODES else torch.float32)
        return dx, None, None, db.to(ctx.bias_dtype) if want_b else None, None


class Mxfp4Linear(torch.nn.Module):
    """A linear layer whose weight is held in 4 bits and frozen, for serving and for training what lies around it (adapters,
    norms, biases): the backward pass gives the input's and the bias's gradients.

    The buffers ``qweight`` and ``scale`` are the weight as the products read it (:class:`PreparedMxfp4Weight`), 17/32 byte a
    weight (of whole 512 columns) and nothing beside them; :meth:`from_weight` makes a layer of a float weight or of a ``(codes, scale)`` pair.
    Activations are bf16, fp16 or fp32. Calls without gradients can be captured into a graph.
    """

    def __init__(self, in_features: int, out_features: int, bias: bool = True, device=None, dtype=None):
        super().__init__()
        self.in_features, self.out_features = in_features, out_features
        self.register_buffer("qweight", torch.zeros(out_features, _row_bytes(in_features), dtype=torch.uint8, device=device))
        self.register_buffer("scale", torch.full((_scale_bytes(out_features, in_features),), 127, dtype=torch.uint8, device=device))
        self.bias = torch.nn.Parameter(torch.zeros(out_features, device=device, dtype=dtype)) if bias else None

    @classmethod
    def from_weight(cls, weight: torch.Tensor, bias: torch.Tensor | None = None, scale: torch.Tensor | None = None,
                    in_features: int | None = None) -> "Mxfp4Linear":
        """The layer of ``weight`` (and ``scale``, ``in_features``: arguments of :func:`prepare_mxfp4_weight`) and ``bias``."""
        form = prepare_mxfp4_weight(weight, scale, in_features)
        layer = cls(form.in_features, form.out_features, bias=False, device="meta")
        layer.qweight, layer.scale = form.q, form.scale
        if bias is not None:
            if bias.shape != (form.out_features,):
                raise ValueError(f"bias of shape {tuple(bias.shape)}, expected ({form.out_features},)")
            with torch.inference_mode(False):
                layer.bias = torch.nn.Parameter(bias.detach().clone())
        return layer

    def prepared(self) -> PreparedMxfp4Weight:
        """The weight for the functions (the buffers themselves)."""
        return PreparedMxfp4Weight(self.qweight, self.scale, self.out_features, self.in_features)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if x.dim() < 1 or x.shape[-1] != self.in_features:
            raise ValueError(f"input of shape {tuple(x.shape)} for a layer of {self.in_features} input features")
        bias = self.bias
        _refuse_tangents(x, bias)
        if not torch.is_grad_enabled() or not (x.requires_grad or (bias is not None and bias.requires_grad)):
            return mxfp4_linear(x, self.prepared(), bias)
        return _Mxfp4LinearFn.apply(x, self.qweight, self.scale, bias, (self.out_features, self.in_features))

    def extra_repr(self) -> str:
        return f"in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}"
