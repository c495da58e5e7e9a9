"""A backward pass of the distillation loss that is recorded without its forward pass, and replayed."""
import pytest
import torch

import graphcuda_b200 as gc
from tests.test_distill_gpu import make

pytestmark = pytest.mark.gpu
DEV = "cuda"
FORMS = [(300, 47, 8), (70, 1000, 8), (160, 9000, 8), (150, 40_001, 8), (40, 5001, 8)]


@pytest.mark.parametrize("M,C,k", FORMS)
def test_replayed_by_itself(M, C, k):
    """What the caller does to the gradient is his affair: a replay writes it again."""
    logits, top, index = make(M, C, k)
    x = logits.detach().requires_grad_()
    (want,) = torch.autograd.grad(gc.distill_loss(x, top, index), x)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream):
        loss = gc.distill_loss(x, top, index)
        stream.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            (dx,) = torch.autograd.grad(loss, x, retain_graph=True)
        for _ in range(2):
            dx.fill_(7)
            graph.replay()
            stream.synchronize()
            assert torch.equal(dx, want)
        dx.fill_(7)
        # the graph of the loss is as it was, for an eager pass too
        (eager,) = torch.autograd.grad(loss, x)
        stream.synchronize()
    assert torch.equal(eager, want) and bool((dx == 7).all())


@pytest.mark.parametrize("M,C,k", FORMS)
def test_forward_and_backward_in_recordings_of_their_own(M, C, k):
    logits, top, index = make(M, C, k)

    class Loss(torch.nn.Module):
        def forward(self, z):
            return gc.distill_loss(z, top, index, None, 2.0, scale=0.1)

    x = logits.detach().requires_grad_()
    want = gc.distill_loss(x, top, index, None, 2.0, scale=0.1)
    (dwant,) = torch.autograd.grad(want, x, torch.tensor(3.0, device=DEV))
    call = torch.cuda.make_graphed_callables(Loss(), (torch.zeros_like(logits).requires_grad_(),))
    for _ in range(2):
        y = logits.detach().requires_grad_()
        got = call(y)
        assert float(got.detach()) == float(want.detach())
        (dgot,) = torch.autograd.grad(got, y, torch.tensor(3.0, device=DEV))
        assert torch.equal(dgot, dwant)
        y = torch.zeros_like(logits).requires_grad_()  # another call between them
        torch.autograd.grad(call(y), y)
