"""Operators whose saved tensors come back from a hook (here: from the host's memory) with other strides than they were saved with."""
import pytest
import torch

import graphcuda_b200 as gc
from tests.test_distill_gpu import make

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("grad", [1.0, -2.0])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M,C,before,behind", [(64, 47, 0, 1), (64, 47, 3, 2), (70, 1000, 0, 3), (160, 9001, 0, 7), (150, 40_001, 1, 6), (40, 5001, 0, 3),
                                               (20, 20_001, 2, 1)])
def test_distill_loss(M, C, before, behind, dtype, grad):
    logits, top, index = make(M, C, 8, seed=C, dtype=dtype)
    wide = torch.zeros(M, before + C + behind, device=DEV, dtype=dtype)
    wide[:, before:before + C] = logits
    x = wide[:, before:before + C].detach().requires_grad_()
    factor = torch.tensor(grad, device=DEV)
    (want,) = torch.autograd.grad(gc.distill_loss(x, top, index, None, 2.0), x, factor)
    with torch.autograd.graph.save_on_cpu():
        loss = gc.distill_loss(x, top, index, None, 2.0)
    for _ in range(2):
        (got,) = torch.autograd.grad(loss, x, factor, retain_graph=True)
        assert torch.equal(got, want)


def test_grouped_linear():
    offsets = torch.tensor([0, 5, 5, 70, 90], dtype=torch.int32, device=DEV)
    x = torch.randn(100, 48, device=DEV).bfloat16()[:, :40].requires_grad_()
    w = torch.randn(4, 40, 40, device=DEV).bfloat16()[:, :, :33].requires_grad_()
    dy = torch.randn(100, 33, device=DEV).bfloat16()
    want = torch.autograd.grad(gc.grouped_linear(x, w, offsets), (x, w), dy)
    with torch.autograd.graph.save_on_cpu():
        y = gc.grouped_linear(x, w, offsets)
    for a, b in zip(torch.autograd.grad(y, (x, w), dy), want):
        assert torch.equal(a, b)
