"""Norm and gated block inside a trace, where more than a first derivative is asked for."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_a_trace_has_no_second_derivative_either(cuda):
    import graphcuda_b200 as gc
    norm, block = gc.RMSNorm(32).to(cuda), gc.GatedFFN(32, 48, 16).to(cuda)
    for module, x in ((norm, torch.randn(5, 32, device=cuda)), (block, torch.randn(5, 32, device=cuda).bfloat16())):
        traced = torch.jit.trace(module, (x,), check_trace=False)
        for f in (module, traced):
            p = next(module.parameters())
            g, = torch.autograd.grad(f(x).float().sum(), p)  # a first one there is
            assert g.any()
            with pytest.raises(RuntimeError, match="derivative|differentiable"):
                g, = torch.autograd.grad(f(x).float().sum(), p, create_graph=True)
                # a penalty on gradient and weights: the gradient's part must not be missing from what comes back
                (g.float().square().sum() + p.float().square().sum()).backward()
