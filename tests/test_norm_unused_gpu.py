"""The norm's backward pass where one of its two outputs is used by nobody."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("traced", [False, True])
@pytest.mark.parametrize("types", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32)], ids=str)
def test_no_gradient_is_made_for_an_unused_stream(cuda, types, traced):
    """Nothing of the matrix' size is allocated but the gradients that are returned."""
    import graphcuda_b200 as gc
    tx, ts = types
    m, n = 20_000, 512
    x, r, w = torch.randn(m, n, device=cuda).to(tx), torch.randn(m, n, device=cuda).to(ts), torch.rand(n, device=cuda) + 0.5
    leaves = [t.requires_grad_() for t in (x, w, r)]
    call = lambda a, b, c: gc.rms_norm(a, b, c)[0]  # noqa: E731
    if traced:
        call = torch.jit.trace(call, tuple(leaves), check_trace=False)
    dy = torch.randn(m, n, device=cuda).to(tx)
    expect = torch.autograd.grad(gc.rms_norm(*leaves), leaves, (dy, torch.zeros(m, n, device=cuda, dtype=ts)))
    y = call(*leaves)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    got = torch.autograd.grad(y, leaves, dy)
    returned = m * n * (x.element_size() + (r.element_size() if ts != tx else 0))
    assert torch.cuda.max_memory_allocated() - before < returned + (4 << 20)
    assert all(a.dtype == b.dtype and torch.equal(a, b) for a, b in zip(got, expect))


def test_an_unused_y(cuda):
    import graphcuda_b200 as gc
    x, r, w = (torch.randn(s, device=cuda).requires_grad_() for s in ((50, 96), (50, 96), (96,)))
    ds = torch.randn(50, 96, device=cuda)
    for call in (lambda a, b, c: gc.rms_norm(a, b, c)[1], torch.jit.trace(lambda a, b, c: gc.rms_norm(a, b, c)[1], (x, w, r),
                                                                          check_trace=False)):
        dx, dw, dr = torch.autograd.grad(call(x, w, r), (x, w, r), ds)
        assert torch.equal(dx, ds) and torch.equal(dr, ds) and not dw.any()
