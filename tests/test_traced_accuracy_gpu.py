"""Predictions and counts inside a trace."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("want", ["pred", "counts", "both", "masks"])
def test_traced_accuracy_runs_on_new_inputs(cuda, want, grad):
    import graphcuda_b200 as gc
    n, c = 501, 7
    labels = torch.randint(0, c, (n,), device=cuda)
    masks = [torch.rand(n, device=cuda) < 0.5 for _ in range(3)]

    def answer(z):
        pred, counts = gc.argmax_accuracy(z, None if want == "pred" else labels, masks if want == "masks" else None,
                                          want_pred=want != "counts")
        return tuple(t for t in (pred, counts) if t is not None)

    with torch.set_grad_enabled(grad):
        zs = [torch.randn(n, c, device=cuda, requires_grad=grad) for _ in range(3)]
        traced = torch.jit.trace(answer, (zs[0],), check_trace=False)
        for z in zs:
            expect = answer(z)
            junk = [torch.full_like(t, -1) for t in expect for _ in range(4)]  # what fresh memory would hold
            del junk
            got = traced(z)
            got = got if isinstance(got, tuple) else (got,)
            assert len(got) == len(expect) and all(torch.equal(a, b) for a, b in zip(got, expect))
