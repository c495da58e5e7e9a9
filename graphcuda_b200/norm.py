"""Root-mean-square norm with the residual's addition, for models deeper than the reference's two layers
(models.ResidualGCN): one kernel forward, one (and the sum of the weight gradient's parts) backward."""
from __future__ import annotations

from typing import Optional

import torch
from torch.nn.parameter import Parameter

from . import _lib

_TYPES = {torch.float32: _lib.TYPE_F32, torch.bfloat16: _lib.TYPE_BF16}


class _TracedNorm(torch.autograd.Function):
    """The norm inside torch.jit.trace (see gcn._TracedConv)."""

    @staticmethod
    def forward(ctx, x, weight, residual, eps, y_type):
        y, stream, saved = _lib.host.rms_norm_forward(x, weight, residual, eps, y_type)
        ctx.save_for_backward(*saved)
        ctx.set_materialize_grads(False)
        ctx.call = y_type, _TYPES[x.dtype], residual is not None
        return y if residual is None else (y, stream)

    @staticmethod
    def backward(ctx, dy, dstream=None):
        if torch.is_grad_enabled():
            raise RuntimeError("rms_norm has no second derivative (create_graph)")
        y_type, x_type, add = ctx.call
        need = ctx.needs_input_grad
        dx, dw, dr = _lib.host.rms_norm_backward(dy, dstream, *ctx.saved_tensors, y_type, x_type, add, need[0] or need[2],
                                                 need[1])
        return dx if need[0] else None, dw, dr if need[2] else None, None, None


class _TracedNormFp8(torch.autograd.Function):
    """The norm with 8-bit rows inside torch.jit.trace."""

    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        y, scale, stream = _lib.host.rms_norm_fp8_forward(x, weight, residual, eps)
        return (y, scale) if residual is None else (y, scale, stream)

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError("rms_norm_fp8 has no gradient: call it under torch.no_grad(), or rms_norm for training")


def rms_norm(x: torch.Tensor, weight: torch.Tensor, residual: Optional[torch.Tensor] = None, eps: float = 1e-6,
             out_dtype: Optional[torch.dtype] = None):
    """``y = h / sqrt(mean(h^2) + eps) * weight`` over the rows of ``h = x + residual``.

    Returns ``y``, or ``(y, h)`` where a residual is given: ``h``, in the residual's type, is the stream that the next
    residual addition continues from.  ``x`` is a float32 or bfloat16 matrix; ``residual`` has its type, or is float32
    beside a bfloat16 ``x``; ``weight`` is float32.  ``out_dtype`` (float32 or bfloat16, default x's) is that of ``y``.
    Statistics are float32, and ``h`` enters them and ``y`` before it is rounded."""
    out = out_dtype or x.dtype
    if out not in _TYPES:
        raise RuntimeError(f"rms_norm: out_dtype must be float32 or bfloat16, got {out} (8 bits: rms_norm_fp8)")
    got = _lib.host.rms_norm(x, weight, residual, eps, _TYPES[out])
    if got is None:
        return _TracedNorm.apply(x, weight, residual, eps, _TYPES[out])
    return got[0] if residual is None else got


def rms_norm_fp8(x: torch.Tensor, weight: torch.Tensor, residual: Optional[torch.Tensor] = None, eps: float = 1e-6):
    """The same norm for serving, with ``y`` in 8 bits: ``(y8, scale)`` or ``(y8, scale, h)``.

    ``y8`` is float8_e4m3fn and stands for ``y8 * scale[:, None]``; a row's scale is its largest |value| / 448 (zero for a
    row of zeros; not finite for a row that holds a NaN or an infinity).  The operand of ``gated_ffn_fp8``."""
    got = _lib.host.rms_norm_fp8(x, weight, residual, eps)
    if got is None:
        return _TracedNormFp8.apply(x, weight, residual, eps)
    return got[:2] if residual is None else got


class RMSNorm(torch.nn.Module):
    """``rms_norm`` with its weight (ones at the start); ``out_dtype`` as there."""

    def __init__(self, width: int, eps: float = 1e-6, out_dtype: Optional[torch.dtype] = None):
        super().__init__()
        self.eps, self.out_dtype = eps, out_dtype
        self.weight = Parameter(torch.ones(width))

    def forward(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None):
        return rms_norm(x, self.weight, residual, self.eps, self.out_dtype)

    def fp8(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None):
        return rms_norm_fp8(x, self.weight, residual, self.eps)
