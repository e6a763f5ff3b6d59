"""Root-mean-square norm behind a residual addition, with outputs that the 8-bit and the 4-bit layer read, and its gradients.

``s = x + residual`` rounded to ``x``'s dtype, ``rstd = 1 / sqrt(E[s^2] + eps)`` with ``eps`` as float32, the mean in float64 and
rounded once to float32, ``y = (s * rstd) * weight`` in float32; ``y`` is rounded once to ``x``'s dtype, or quantized. The norm under the
reference's rms_adaln (h3serve/native_engine/model/kernels.py:7594-7640), with a learned weight in place of the modulation.

Every function runs the HIP kernels of libmx_qlinear.so on the tensors' GPU and current stream; there is no CPU path.
"""

from __future__ import annotations

import torch

from . import _lib
from . import fp8, mxfp4
from .fp8 import _float_code, _norm_params, _refuse_capture, _refuse_tangents, _room, _rows_in_place, _view, _workspace
from .ops import _launch, _ptr, _require_gpu, _vector


def _rms(what: str, x: torch.Tensor, weight, eps: float, residual, want_rstd: bool, target: int | None):
    """The forward pass: (y or the pair's storage as a tuple, [sum], [rstd])."""
    code = _float_code(x, "input")
    if x.dim() < 1 or x.shape[-1] == 0:
        raise ValueError(f"{what} needs a non-empty last dimension")
    if not eps >= 0:
        raise ValueError(f"eps must not be negative, got {eps}")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype):
        raise ValueError(f"residual of {residual.dtype} {tuple(residual.shape)} for an input of {x.dtype} {tuple(x.shape)}")
    dev = _require_gpu(x, residual, weight)
    flat, d = x.dim() == 2, x.shape[-1]
    w, _, pcode = _norm_params(d, dev, x.dtype, weight, None, "rms norm")
    x2 = _rows_in_place(x, d)
    m = x2.shape[0]
    ldx, r2, ldr, total = x2.stride(0) if m > 1 else d, None, 0, None
    if residual is not None:
        r2 = _rows_in_place(residual, d)
        ldr, total = r2.stride(0) if m > 1 else d, torch.empty(m, d, dtype=x.dtype, device=dev)
    rstd = torch.empty(m, dtype=torch.float32, device=dev) if want_rstd else None
    if target is None:
        y, s, target, lds = torch.empty(m, d, dtype=x.dtype, device=dev), None, code, 0
    else:
        y, s = fp8._new_pair(m, d, dev) if target == _lib.DTYPE_E4M3 else mxfp4._new_pair(m, d, dev)
        lds = s.shape[1]
    if m:
        _launch(dev, "mxq_rms_norm", x2.data_ptr(), _ptr(r2), code, ldx, ldr, _ptr(w), pcode, float(eps), _ptr(total), y.data_ptr(),
                target, y.shape[1], _ptr(s), lds, _ptr(rstd), m, d)
    rest = []
    if total is not None:
        rest.append(total if flat else total.reshape(x.shape))
    if want_rstd:
        rest.append(rstd if flat else rstd.reshape(x.shape[:-1]))
    return (y, s), rest


def rms_norm(x: torch.Tensor, weight: torch.Tensor | None = None, eps: float = 1e-5, residual: torch.Tensor | None = None,
             return_rstd: bool = False):
    """``y = s * rstd * weight`` over the last dimension (at most 24576) with ``s = x + residual`` (``s = x`` without one); ``eps``
    counts as float32 (1e-5: 9.99999975e-6).
    Returns ``y``; with ``residual`` also ``s``, the residual stream behind the addition, and with ``return_rstd`` the rows'
    float32 ``rstd``, which :func:`rms_norm_backward` takes: ``(y[, s][, rstd])``."""
    (y, _), rest = _rms("rms_norm", x, weight, eps, residual, return_rstd, None)
    y = y if x.dim() == 2 else y.reshape(x.shape)
    return (y, *rest) if rest else y


def rms_norm_quantize_fp8(x: torch.Tensor, weight: torch.Tensor | None = None, eps: float = 1e-5,
                          residual: torch.Tensor | None = None, return_rstd: bool = False):
    """:func:`rms_norm` with ``y`` quantized from float32 as :func:`quantize_fp8_block128` does: ``(codes, scale[, s][, rstd])``,
    a pair for :func:`fp8_linear_prequantized` in one launch."""
    (q, s), rest = _rms("rms_norm_quantize_fp8", x, weight, eps, residual, return_rstd, _lib.DTYPE_E4M3)
    lead, d = tuple(x.shape[:-1]), x.shape[-1]
    return (_view(q, lead, d), _view(s, lead, -(-d // fp8.BLOCK)), *rest)


def rms_norm_quantize_mxfp4(x: torch.Tensor, weight: torch.Tensor | None = None, eps: float = 1e-5,
                            residual: torch.Tensor | None = None, return_rstd: bool = False):
    """:func:`rms_norm` with ``y`` quantized from float32 as :func:`quantize_mxfp4` does: ``(codes, scale[, s][, rstd])``, a pair
    for :func:`mxfp4_linear_prequantized` in one launch (of more than 16 rows, or fewer of a long ``K``, each product lays the
    scales out for itself first, and copies the codes where ``K`` is not a multiple of 256)."""
    (q, s), rest = _rms("rms_norm_quantize_mxfp4", x, weight, eps, residual, return_rstd, _lib.DTYPE_E2M1)
    return (*mxfp4._as_pair(q, s, tuple(x.shape[:-1]), x.shape[-1]), *rest)


def rms_norm_backward(dy: torch.Tensor, x, rstd: torch.Tensor, weight: torch.Tensor | None = None,
                      dsum: torch.Tensor | None = None, needs_params: bool = True):
    """Gradients ``(dx, dweight)`` of :func:`rms_norm`: ``dx`` in ``dy``'s dtype, that of ``x`` and of ``residual`` alike,
    ``dweight`` in float32 (``None`` without ``needs_params``). ``x`` is what was normed (the forward's ``s`` where a residual
    was added), or that as it was kept in 8 bits, a ``(codes, scale)`` pair of :func:`quantize_fp8_block128`; ``rstd`` is the
    forward's, and ``dsum`` the gradient that reaches ``s`` beside the norm, which is added."""
    code = _float_code(dy, "gradient")
    if dy.dim() < 1 or dy.shape[-1] == 0:
        raise ValueError("rms_norm_backward needs a non-empty last dimension")
    d = dy.shape[-1]
    if isinstance(x, (tuple, list)):
        if tuple(x[0].shape) != tuple(dy.shape):
            raise ValueError(f"input of shape {tuple(x[0].shape)} for a gradient of shape {tuple(dy.shape)}")
        x2, xs, _, _ = fp8._pair(*x)
        xcode, ldxs = _lib.DTYPE_E4M3, max(xs.stride(0), xs.shape[1])
    else:
        if tuple(x.shape) != tuple(dy.shape):
            raise ValueError(f"input of shape {tuple(x.shape)} for a gradient of shape {tuple(dy.shape)}")
        if x.dtype != dy.dtype:
            raise ValueError(f"input of {x.dtype} for a gradient of {dy.dtype}")
        x2, xs, xcode, ldxs = _rows_in_place(x, d), None, code, 0
    if dsum is not None and (dsum.shape != dy.shape or dsum.dtype != dy.dtype):
        raise ValueError(f"gradient of the sum of {dsum.dtype} {tuple(dsum.shape)} for a gradient of {dy.dtype} {tuple(dy.shape)}")
    y2 = _rows_in_place(dy, d)
    m = y2.shape[0]
    if rstd.dtype != torch.float32 or rstd.numel() != m:
        raise ValueError(f"rstd must be float32 with one entry per row ({m}), got {rstd.dtype} {tuple(rstd.shape)}")
    dev = _require_gpu(dy, x2, xs, rstd, weight, dsum)
    w, _, pcode = _norm_params(d, dev, dy.dtype, weight, None, "rms norm")
    s2 = None if dsum is None else _rows_in_place(dsum, d)
    dx = torch.empty(m, d, dtype=dy.dtype, device=dev)
    dw = torch.empty(d, dtype=torch.float32, device=dev) if needs_params else None
    need = _workspace("mxq_rms_norm_backward_workspace", dev.index, m, d) if needs_params else 0
    ws = _room(need, dev)
    if m or needs_params:
        rstd = _vector(rstd, torch.float32, dev)
        _launch(dev, "mxq_rms_norm_backward", y2.data_ptr(), code, max(y2.stride(0), d), x2.data_ptr(), xcode, max(x2.stride(0), d),
                _ptr(xs), ldxs, rstd.data_ptr(), _ptr(w), pcode, _ptr(s2), 0 if s2 is None else max(s2.stride(0), d), dx.data_ptr(),
                _ptr(dw), m, d, _ptr(ws), need)
    return dx if dy.dim() == 2 else dx.reshape(dy.shape), dw


class _RMSNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, eps, keep_fp8):
        _refuse_capture(x.device)
        ctx.set_materialize_grads(False)
        out = rms_norm(x, weight, eps, residual, return_rstd=True)
        s, rstd = (x if residual is None else out[1]), out[-1]
        kept = fp8.quantize_fp8_block128(s) if keep_fp8 else (s,)
        ctx.save_for_backward(rstd, weight, *kept)
        return out[0] if residual is None else out[:2]

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, ds=None):
        rstd, weight, *kept = ctx.saved_tensors
        want_x, want_r, want_w = ctx.needs_input_grad[:3]
        if dy is None:  # (the norm's own output was not used)
            return (ds if want_x else None), (ds if want_r else None), None, None, None
        _refuse_capture(dy.device)
        x = tuple(kept) if len(kept) == 2 else kept[0]
        dx, dw = rms_norm_backward(dy, x, rstd, weight, ds, needs_params=want_w)
        return (dx if want_x else None), (dx if want_r else None), dw.to(weight.dtype) if want_w else None, None, None


class RMSNorm(torch.nn.Module):
    """Root-mean-square norm over the last dimension (:func:`rms_norm`) with a learned weight: ``norm(x)`` gives ``y``,
    ``norm(x, residual)`` the pair ``(y, x + residual)``. ``keep_fp8`` keeps what is normed for the backward pass in 8 bits
    instead of as it is."""

    def __init__(self, features: int, eps: float = 1e-5, keep_fp8: bool = False, device=None, dtype=None):
        super().__init__()
        self.features, self.eps, self.keep_fp8 = features, eps, keep_fp8
        self.weight = torch.nn.Parameter(torch.ones(features, device=device, dtype=dtype))

    def forward(self, x: torch.Tensor, residual: torch.Tensor | None = None):
        if x.dim() < 1 or x.shape[-1] != self.features:
            raise ValueError(f"input of shape {tuple(x.shape)} for a norm of {self.features} features")
        weight = self.weight
        _refuse_tangents(x, residual, weight)
        if not torch.is_grad_enabled() or not (x.requires_grad or weight.requires_grad or (residual is not None and residual.requires_grad)):
            return rms_norm(x, weight, self.eps, residual)
        return _RMSNormFn.apply(x, residual, weight, self.eps, self.keep_fp8)

    def extra_repr(self) -> str:
        return f"{self.features}, eps={self.eps}, keep_fp8={self.keep_fp8}"
