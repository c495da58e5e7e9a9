"""The stacked model of the reference's training script
(tests/gcn/graphcuda_impl.py:15-24), generalised to any depth: GCNConv layers
with ReLU on all but the last, ``log_softmax`` on top."""
from __future__ import annotations

import copy
from typing import Optional, Sequence

import torch

from .ffn import GatedFFN
from .gcn import GCNConv
from .losses import argmax_accuracy
from .norm import RMSNorm


class GCN(torch.nn.Module):
    def __init__(self, dims: Sequence[int], *, precision: Optional[str] = None, fuse_relu_backward: bool = True):
        super().__init__()
        self.convs = torch.nn.ModuleList(
            [GCNConv(dims[i], dims[i + 1], apply_relu=(i < len(dims) - 2), precision=precision)
             for i in range(len(dims) - 1)])
        if fuse_relu_backward:
            # Layer i's ReLU output has exactly one consumer here (layer i + 1), so the ReLU backward of layer i
            # is applied where layer i + 1 produces its input gradient (reference gcn.cu:36 as a fused store).
            for lower, upper in zip(self.convs[:-1], self.convs[1:]):
                if lower.apply_relu:
                    lower.fuse_relu_backward |= 1
                    upper.fuse_relu_backward |= 2

    def forward(self, x, adj, log_softmax: bool = True, return_hidden: bool = False):
        """log_softmax=False returns the last layer's raw output, for
        losses.log_softmax_nll_loss which fuses the normalisation with the loss.
        return_hidden=True returns (output, [x, h1, ..., logits]): every layer's
        input and output, for checks that compare layer by layer."""
        hidden = [x]
        for conv in self.convs:
            x = conv(x, adj)
            hidden.append(x)
        out = torch.log_softmax(x, dim=1) if log_softmax else x
        return (out, hidden) if return_hidden else out

    @torch.no_grad()
    def evaluate(self, x, adj, labels, masks=None):
        """The reference script's ``test()`` (tests/gcn/graphcuda_impl.py:60-69): a forward pass without
        autograd state (nothing is saved, no mask is written, log_softmax is skipped because it does not
        move the argmax) followed by the fused argmax / count kernel.  Returns ``(pred, counts)`` as
        losses.argmax_accuracy does; ``(counts[:, 0] / counts[:, 1]).tolist()`` gives the accuracies with
        one host read."""
        return argmax_accuracy(self.forward(x, adj, log_softmax=False), labels, masks)


class ResidualBlock(torch.nn.Module):
    """One layer of ResidualGCN on its float32 stream: norm, graph layer, norm, gated feed-forward block.

    Every addition to the stream happens inside the norm that reads it next: ``forward(y, h)`` takes the stream and what
    the block before adds to it (None at first) and returns the stream and this block's own addition."""

    def __init__(self, width: int, hidden: int, activation: str = "silu", precision: Optional[str] = None):
        super().__init__()
        self.norm_conv = RMSNorm(width, out_dtype=torch.float32)
        self.conv = GCNConv(width, width, apply_relu=False, precision=precision)
        self.norm_ffn = RMSNorm(width, out_dtype=torch.bfloat16)
        self.ffn = GatedFFN(width, hidden, width, activation)

    def aggregate(self, y, h, adj):
        n, h = (self.norm_conv(h), h) if y is None else self.norm_conv(y, h)
        return self.conv(n, adj), h

    def forward(self, y, h, adj):
        a, h = self.aggregate(y, h, adj)
        n, h = self.norm_ffn(a, h)
        return self.ffn(n), h


class ResidualGCN(torch.nn.Module):
    """A deep GCN: ``layers`` residual blocks of ``width`` between an input and an output graph layer.

    Graph layers run in float32 (or ``precision``), feed-forward blocks in bfloat16 with bfloat16 weights, of which
    optim.FusedAdamW keeps float32 masters.  Interchangeable with ``GCN`` for graphed.GraphedTrainStep and ``evaluate``."""

    def __init__(self, in_dim: int, width: int, layers: int, classes: int, *, hidden: Optional[int] = None,
                 activation: str = "silu", precision: Optional[str] = None):
        super().__init__()
        self.conv_in = GCNConv(in_dim, width, apply_relu=False, precision=precision)
        self.blocks = torch.nn.ModuleList(
            [ResidualBlock(width, hidden or 4 * width, activation, precision) for _ in range(layers)])
        self.norm_out = RMSNorm(width, out_dtype=torch.float32)
        self.conv_out = GCNConv(width, classes, apply_relu=False, precision=precision)

    def _blocks(self, y, h, adj):
        for block in self.blocks:
            y, h = block(y, h, adj)
        return y, h

    def forward(self, x, adj, log_softmax: bool = True):
        """``log_softmax=False`` returns the output layer's raw logits, for losses.log_softmax_nll_loss."""
        y, h = self._blocks(None, self.conv_in(x, adj), adj)
        n = self.norm_out(h) if y is None else self.norm_out(y, h)[0]
        out = self.conv_out(n, adj)
        return torch.log_softmax(out, dim=1) if log_softmax else out

    @torch.no_grad()
    def evaluate(self, x, adj, labels, masks=None):
        """As ``GCN.evaluate``: ``(pred, counts)``."""
        return argmax_accuracy(self.forward(x, adj, log_softmax=False), labels, masks)

    def for_serving(self, bits: int = 8) -> "ServedResidualGCN":
        """The model with the first product of every feed-forward block in 8 bits, or with all weights of these blocks in 4; its
        weights are those of this moment."""
        return ServedResidualGCN(self, bits)


def _frozen(module: torch.nn.Module) -> torch.nn.Module:
    return copy.deepcopy(module).requires_grad_(False)


class ServedBlock(ResidualBlock):
    """``ResidualBlock`` with its feed-forward block in 8 or 4 bits: weights of their own, those that the block had."""

    bits = 8  # what blocks have that were pickled when there was no choice

    def __init__(self, block: ResidualBlock, bits: int = 8):
        torch.nn.Module.__init__(self)
        self.norm_conv, self.conv, self.norm_ffn = (_frozen(m) for m in (block.norm_conv, block.conv, block.norm_ffn))
        self.ffn = block.ffn.for_serving(bits)
        self.bits = bits

    def forward(self, y, h, adj):
        if self.bits == 4:
            return super().forward(y, h, adj)
        a, h = self.aggregate(y, h, adj)
        n8, scale, h = self.norm_ffn.fp8(a, h)
        return self.ffn(n8, scale), h


class ServedResidualGCN(ResidualGCN):
    """``ResidualGCN`` for inference.  ``bits=8``: the norm in front of a feed-forward block writes 8 bits and a scale per row, which
    the block multiplies with weights laid out in 8 bits once.  ``bits=4``: both weights of every feed-forward block have 4 bits.
    All of its weights are copies: the source may train on, or go."""

    bits = 8  # as in ServedBlock

    def __init__(self, model: ResidualGCN, bits: int = 8):
        torch.nn.Module.__init__(self)
        self.bits = bits
        self.conv_in, self.norm_out, self.conv_out = (_frozen(m) for m in (model.conv_in, model.norm_out, model.conv_out))
        self.blocks = torch.nn.ModuleList([ServedBlock(block, bits) for block in model.blocks])

    def for_serving(self, bits: Optional[int] = None) -> "ServedResidualGCN":
        if bits not in (None, self.bits):
            raise RuntimeError(f"the model serves in {self.bits} bits: ask the one that it was made of")
        return self

    @torch.no_grad()
    def forward(self, x, adj, log_softmax: bool = True):
        return super().forward(x, adj, log_softmax)
