"""Weights per kind of row: products of rows that are sorted by group, for graphs whose vertices are of several kinds."""
from __future__ import annotations

import math

import torch
from torch.nn.parameter import Parameter

from . import _lib


class _TracedGrouped(torch.autograd.Function):
    """The product inside torch.jit.trace (see gcn._TracedConv)."""

    @staticmethod
    def forward(ctx, x, w, offsets):
        y, saved = _lib.host.grouped_linear_forward(x, w, offsets)
        ctx.save_for_backward(*saved)
        return y

    @staticmethod
    def backward(ctx, dy):
        if torch.is_grad_enabled():
            raise RuntimeError("grouped_linear has no second derivative (create_graph)")
        return _lib.host.grouped_linear_backward(dy, *ctx.saved_tensors, *ctx.needs_input_grad[:2]) + (None,)


def grouped_linear(x: torch.Tensor, w: torch.Tensor, offsets: torch.Tensor) -> torch.Tensor:
    """``y[r] = x[r] @ w[g]`` for the rows of every group g, ``offsets[g] <= r < offsets[g + 1]``.

    ``x`` is [rows, in] with its rows sorted by group, ``w`` [groups, in, out], both bfloat16, as is the result; ``offsets`` is
    int32 [groups + 1] on the device, like a CSR's row pointers, and is not read by the host.  Groups may be empty.  Rows before
    the first offset and from the last one on belong to no group: their results, and their gradients, are zeros.
    Sums are float32, rounded once.  Widths that are multiples of 8 are read in place, others through padded copies."""
    y = _lib.host.grouped_linear(x, w, offsets)
    return y if y is not None else _TracedGrouped.apply(x, w, offsets)


class GroupedLinear(torch.nn.Module):
    """``grouped_linear`` with its weights, bfloat16 (optim.FusedAdamW keeps float32 masters of such)."""

    def __init__(self, in_dim: int, out_dim: int, groups: int):
        super().__init__()
        self.weight = Parameter((torch.randn(groups, in_dim, out_dim) / math.sqrt(max(in_dim, 1))).bfloat16())

    def forward(self, x: torch.Tensor, offsets: torch.Tensor) -> torch.Tensor:
        return grouped_linear(x, self.weight, offsets)
