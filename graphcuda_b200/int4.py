"""Weights of 4 bits for serving: laid out once, multiplied by the rows of a call (models.ServedResidualGCN with bits=4)."""
from __future__ import annotations

from typing import Optional

import torch

from . import _lib
from .ffn import _act

GROUPS = (32, 64, 128)
_CHUNK = 128  # inputs whose codes lie together


class Int4Weight(torch.nn.Module):
    """A weight matrix [in, out] of 4-bit codes: ``(code - zero) * scale`` with a bfloat16 scale, and a zero point of 0 to 15 (8 where
    there is none), for every ``group`` inputs of an output.  Made by ``quantize_weight_int4`` or, of codes that exist, by
    ``from_codes``; ``dequantize`` gives the values back.  Its buffer is in the order in which the kernels read it."""

    def __init__(self, records: torch.Tensor, zero_points: bool, in_features: int, out_features: int, group: int):
        super().__init__()
        self.zero_points, self.in_features, self.out_features, self.group = zero_points, in_features, out_features, group
        # uint8 [out / 16, in / 128, record]: codes [16, 64], scales [16, 128 / group] of 2 bytes, zero points [16, 128 / group] of one
        self.register_buffer("records", records)

    @staticmethod
    def from_codes(codes: torch.Tensor, scale: torch.Tensor, zero: Optional[torch.Tensor] = None, *, group: int) -> "Int4Weight":
        """``codes`` is uint8 [in, out] with values 0 to 15; ``scale`` bfloat16 and ``zero`` uint8 (0 to 15, or None) are
        [ceil(in / group), out]: input k belongs to group ``k // group``, of 32, 64 or 128."""
        if group not in GROUPS:
            raise RuntimeError(f"Int4Weight: a group is one of {GROUPS} inputs, got {group}")
        if codes.dim() != 2 or codes.dtype != torch.uint8:
            raise RuntimeError("Int4Weight: codes must be a uint8 matrix [in, out]")
        k, n = codes.shape
        groups = -(-k // group)
        if scale.shape != (groups, n) or scale.dtype != torch.bfloat16 or scale.device != codes.device:
            raise RuntimeError("Int4Weight: scale must be bfloat16 [ceil(in / group), out] on the codes' device")
        if zero is not None and (zero.shape != (groups, n) or zero.dtype != torch.uint8 or zero.device != codes.device):
            raise RuntimeError("Int4Weight: zero must be uint8 [ceil(in / group), out] on the codes' device")
        for what in (codes, zero):
            if what is not None and what.numel() and int(what.max()) > 15:
                raise RuntimeError("Int4Weight: codes and zero points are 0 to 15")
        blocks, chunks, per = -(-n // 16), -(-k // _CHUNK), _CHUNK // group
        if k % _CHUNK or n % 16:
            codes = torch.nn.functional.pad(codes, (0, blocks * 16 - n, 0, chunks * _CHUNK - k))
        # inputs: chunk, 32s, lane, and the four codes of either half of a lane's word, two to a byte; outputs: block, row
        q = codes.reshape(chunks, 4, 4, 2, 2, 2, blocks, 16)
        q = q[:, :, :, :, 0] | q[:, :, :, :, 1] << 4
        records = codes.new_empty(blocks, chunks, 1024 + 16 * per * (2 if zero is None else 3))
        records[..., :1024].view(blocks, chunks, 16, 4, 4, 2, 2).copy_(q.permute(5, 0, 6, 2, 1, 4, 3))

        def lay(t, at):
            s = t.new_zeros(blocks * 16, chunks * per)
            s[:n, :groups] = t.t()
            s = s.view(blocks, 16, chunks, per).transpose(1, 2).contiguous().view(blocks, chunks, 16 * per).view(torch.uint8)
            records[..., at:at + s.size(2)] = s

        lay(scale, 1024)
        if zero is not None:
            lay(zero, 1024 + 32 * per)
        return Int4Weight(records, zero is not None, k, n, group)

    def dequantize(self) -> torch.Tensor:
        """The weights' values, float32 [in, out]."""
        blocks, chunks = self.records.shape[:2]
        per = _CHUNK // self.group
        codes, scale, zero = self.records.split((1024, 32 * per, 16 * per if self.zero_points else 0), 2)
        q = torch.stack((codes & 15, codes >> 4), -1).view(blocks, chunks, 2, 8, 4, 4, 2, 4)
        q = q.permute(0, 2, 3, 1, 5, 4, 7, 6).reshape(blocks * 16, chunks * _CHUNK)

        def flat(t):
            t = t.reshape(blocks, chunks, 16, per).transpose(1, 2).reshape(blocks * 16, chunks * per)
            return t.repeat_interleave(self.group, 1).float()

        w = (q.float() - (flat(zero) if self.zero_points else 8.0)) * flat(scale.contiguous().view(torch.bfloat16))
        return w[:self.out_features, :self.in_features].t().contiguous()

    def _parts(self):
        return self.records, self.zero_points, self.group, self.in_features, self.out_features

    def extra_repr(self) -> str:
        return f"in_features={self.in_features}, out_features={self.out_features}, group={self.group}, zero_points={self.zero_points}"


def quantize_weight_int4(w: torch.Tensor, group: int = 64, zero_points: bool = False) -> Int4Weight:
    """``w`` [in, out] in 4 bits, for ``linear_int4`` and ``gated_ffn_int4``.  Every ``group`` inputs (32, 64 or 128) of an output
    share a scale: their largest |value| / 7.5, or with ``zero_points`` the width of their range (zero in it) / 15.  Laid out
    once, by whoever serves the model."""
    if w.dim() != 2 or not w.is_floating_point():
        raise RuntimeError("quantize_weight_int4: a matrix of floating-point weights expected")
    if group not in GROUPS:
        raise RuntimeError(f"quantize_weight_int4: a group is one of {GROUPS} inputs, got {group}")
    w = w.detach().float()
    if not bool(w.isfinite().all()):
        raise RuntimeError("quantize_weight_int4: weights must be finite")
    k, n = w.shape
    groups = -(-k // group)
    t = w.new_zeros(groups * group, n)
    t[:k] = w
    t = t.view(groups, group, n)
    if zero_points:
        low, high = t.amin(1).clamp(max=0), t.amax(1).clamp(min=0)  # (the zeros that fill the last group up are in that range)
        scale = (high / 15 - low / 15).bfloat16()
        step = torch.where(scale > 0, scale, 1.0).float()
        zero = (-low / step).round().clamp(0, 15)
    else:
        scale = (t.abs().amax(1) / 7.5).bfloat16()
        step = torch.where(scale > 0, scale, 1.0).float()
        zero = torch.full_like(step, 8)
    codes = (t / step[:, None] + zero[:, None]).round().clamp(0, 15).to(torch.uint8).view(groups * group, n)[:k]
    return Int4Weight.from_codes(codes, scale, zero.to(torch.uint8) if zero_points else None, group=group)


class _TracedLinear(torch.autograd.Function):
    """The product inside torch.jit.trace (see gcn._TracedConv)."""

    @staticmethod
    def forward(ctx, x, *call):
        return _lib.host.linear_int4_forward(x, *call)

    @staticmethod
    def backward(ctx, dy):
        raise RuntimeError("linear_int4 has no gradient: call it under torch.no_grad()")


class _TracedBlock(torch.autograd.Function):
    """The block inside torch.jit.trace."""

    @staticmethod
    def forward(ctx, x, *call):
        return _lib.host.gated_ffn_int4_forward(x, *call)

    @staticmethod
    def backward(ctx, dy):
        raise RuntimeError("gated_ffn_int4 has no gradient: call it under torch.no_grad(), or gated_ffn for training")


def linear_int4(x: torch.Tensor, w: Int4Weight) -> torch.Tensor:
    """``x @ w``: ``x`` is bfloat16 [rows, in], the result bfloat16 [rows, out], sums are float32.

    Up to 128 rows the weights' values enter unrounded, and only the result's rounding shows.  For more rows they are rounded to
    bfloat16 on their way to the tensor cores, which adds as much again (2.4e-3 instead of 1.7e-3, relative, root mean square), and take
    two bytes each in the call's own memory."""
    y = _lib.host.linear_int4(x, *w._parts())
    return y if y is not None else _TracedLinear.apply(x, *w._parts())


def gated_ffn_int4(x: torch.Tensor, w_in: Int4Weight, w_out: Int4Weight, activation: str = "silu") -> torch.Tensor:
    """``gated_ffn`` for serving with both weights in 4 bits: ``(act(x @ Wg) * (x @ Wu)) @ w_out`` with ``w_in = [Wg | Wu]``; ``x``
    and the result are bfloat16.

    Up to 64 rows nothing is rounded on the way but the result.  For more rows the weights and the hidden row between the products are
    rounded to 11 bits, an eighth of the result's own rounding: they and ``x`` are held in fp16 with powers of two per output and row.  What
    keeps fewer bits is a value of ``x`` below 2^-28 of its row's largest, a group of weights below 2^-23 of its output's largest, and a
    hidden value below 2^-13 of its row's largest (columns whose weights are larger than others' by a factor of up to 2^14 are taken down
    by it first)."""
    act = _act(activation)
    y = _lib.host.gated_ffn_int4(x, *w_in._parts(), *w_out._parts(), act)
    return y if y is not None else _TracedBlock.apply(x, *w_in._parts(), *w_out._parts(), act)


class GatedFFNInt4(torch.nn.Module):
    """A ``GatedFFN`` for inference with its weights, of this moment, in 4 bits."""

    def __init__(self, block: torch.nn.Module, group: int = 64, zero_points: bool = False):
        super().__init__()
        self.activation = block.activation
        self.w_in = quantize_weight_int4(block.w_in, group, zero_points)
        self.w_out = quantize_weight_int4(block.w_out, group, zero_points)

    @torch.no_grad()
    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return gated_ffn_int4(x, self.w_in, self.w_out, self.activation)
