"""Gated feed-forward block, applied to every vertex between two aggregations (models.ResidualGCN): bf16 on the tensor
cores, both projections, the activation and their product in one kernel, the second product in another; for serving,
the first product in 8 bits."""
from __future__ import annotations

import math

import torch
from torch.nn.parameter import Parameter

from . import _lib

ACTIVATIONS = {"silu": _lib.ACT_SILU, "gelu": _lib.ACT_GELU, "relu": _lib.ACT_RELU}


def _act(name: str) -> int:
    try:
        return ACTIVATIONS[name]
    except KeyError:
        raise ValueError(f"activation must be one of {sorted(ACTIVATIONS)}, got {name!r}") from None


class _TracedFFN(torch.autograd.Function):
    """The block inside torch.jit.trace (see gcn._TracedConv)."""

    @staticmethod
    def forward(ctx, x, w_in, w_out, act):
        y, saved = _lib.host.gated_ffn_forward(x, w_in, w_out, act)
        ctx.save_for_backward(*saved)
        ctx.act = act
        return y

    @staticmethod
    def backward(ctx, dy):
        if torch.is_grad_enabled():
            raise RuntimeError("gated_ffn has no second derivative (create_graph)")
        return _lib.host.gated_ffn_backward(dy, *ctx.saved_tensors, ctx.act, *ctx.needs_input_grad[:3]) + (None,)


class _TracedFFNFp8(torch.autograd.Function):
    """The block with its first product in 8 bits inside torch.jit.trace."""

    @staticmethod
    def forward(ctx, x8, x_scale, w8, w_scale, w_out, act):
        return _lib.host.gated_ffn_fp8_forward(x8, x_scale, w8, w_scale, w_out, act)

    @staticmethod
    def backward(ctx, dy):
        raise RuntimeError("gated_ffn_fp8 has no gradient: call it under torch.no_grad(), or gated_ffn for training")


def gated_ffn(x: torch.Tensor, w_in: torch.Tensor, w_out: torch.Tensor, activation: str = "silu") -> torch.Tensor:
    """``(act(x @ Wg) * (x @ Wu)) @ w_out`` with ``w_in = [Wg | Wu]``, all bfloat16.

    ``x`` is [rows, in], ``w_in`` [in, 2 * hidden], ``w_out`` [hidden, out] (in x out, like GCNConv's weights).  Sums are
    float32.  Of more than 64 rows the hidden row is rounded to bfloat16 before the second product, and so is the gradient of
    ``x @ w_in`` in the backward pass: results are off by 2.4e-3 (relative, root mean square), of which the output's own rounding is
    1.7e-3.  Of 64 rows and fewer both are kept to 16 bits and more, and only the output's rounding shows; so a row's result in a
    large call differs from that in a small one by as much.  ``x @ w_in`` itself is kept for the backward pass to 11 bits, with an
    exponent for every 32 columns of a row.
    ``activation``: "silu", "gelu" (with erf) or "relu".  Widths that are multiples of 8 are read in place, others through
    padded copies."""
    act = _act(activation)
    y = _lib.host.gated_ffn(x, w_in, w_out, act)
    return y if y is not None else _TracedFFN.apply(x, w_in, w_out, act)


def quantize_weight_fp8(w: torch.Tensor):
    """``(w8, scale)`` for ``gated_ffn_fp8``: w is [in, out]; w8 is float8_e4m3fn [out, in] and stands for
    ``w8[n] * scale[n]``, scale[n] being the column's largest |value| / 448.  Laid out once, by whoever serves the model."""
    if w.dim() != 2 or not w.is_floating_point():
        raise RuntimeError("quantize_weight_fp8: a matrix of floating-point weights expected")
    wt = w.detach().float().t()
    scale = wt.abs().amax(1) / 448.0 if w.size(0) else wt.new_zeros(wt.size(0))
    # of a scale that is subnormal, and so rounded coarsely, there may be more than 448 in the largest value, which has no code
    q = (wt / torch.where(scale > 0, scale, 1.0)[:, None]).clamp(-448.0, 448.0)
    return q.contiguous().to(torch.float8_e4m3fn), scale


def gated_ffn_fp8(x8: torch.Tensor, x_scale: torch.Tensor, w_in8: torch.Tensor, w_in_scale: torch.Tensor,
                  w_out: torch.Tensor, activation: str = "silu") -> torch.Tensor:
    """The block for serving, its first product in 8 bits: ``x8, x_scale`` as ``rms_norm_fp8`` leaves them,
    ``w_in8, w_in_scale`` from ``quantize_weight_fp8``; ``w_out`` and the result are bfloat16, and the hidden row between the
    products is rounded as in ``gated_ffn``."""
    act = _act(activation)
    y = _lib.host.gated_ffn_fp8(x8, x_scale, w_in8, w_in_scale, w_out, act)
    return y if y is not None else _TracedFFNFp8.apply(x8, x_scale, w_in8, w_in_scale, w_out, act)


class GatedFFN(torch.nn.Module):
    """``gated_ffn`` with its weights, bfloat16 (optim.FusedAdamW keeps float32 masters of such)."""

    def __init__(self, in_dim: int, hidden: int, out_dim: int, activation: str = "silu"):
        super().__init__()
        _act(activation)
        self.activation = activation
        self.w_in = Parameter((torch.randn(in_dim, 2 * hidden) / math.sqrt(max(in_dim, 1))).bfloat16())
        self.w_out = Parameter((torch.randn(hidden, out_dim) / math.sqrt(max(hidden, 1))).bfloat16())

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return gated_ffn(x, self.w_in, self.w_out, self.activation)

    def for_serving(self) -> "GatedFFNFp8":
        """The block with its first product in 8 bits; its weights are those of this moment."""
        return GatedFFNFp8(self)


class GatedFFNFp8(torch.nn.Module):
    def __init__(self, block: GatedFFN):
        super().__init__()
        self.activation = block.activation
        w8, scale = quantize_weight_fp8(block.w_in)
        self.register_buffer("w_in8", w8)
        self.register_buffer("w_in_scale", scale)
        self.register_buffer("w_out", block.w_out.detach().clone())

    @torch.no_grad()
    def forward(self, x8: torch.Tensor, x_scale: torch.Tensor) -> torch.Tensor:
        return gated_ffn_fp8(x8, x_scale, self.w_in8, self.w_in_scale, self.w_out, self.activation)
