"""What a grouped product asks for as workspace: copies only of operands that cannot be read in place."""
import pytest
import torch

import graphcuda_b200 as gc
from graphcuda_b200 import _lib

L = _lib.lib


def need(m, k, n, g, dx=0, dw=0, dy=16, lddy=None, x=16, ldx=None, w=16, ldw=None):
    return L().gc_grouped_linear_workspace_bytes_for(dy, lddy or n, x, ldx or k, w, ldw or n, m, k, n, g, dx, dw)


def test_aligned_operands_need_no_copies():
    for m, k, n, g in ((16_384, 2048, 4096, 16), (64, 4096, 4096, 128)):
        assert need(m, k, n, g) <= 4096 and need(m, k, n, g, dx=1) <= 4096
        # the rows that fill up no block of 64, and fp32 parts of dW, for which there is no other place
        tails = g * 64 * (k + n) * 2
        parts = 4 * k * n * (m // 1024 + g)
        assert need(m, k, n, g, dw=1) <= tails + parts + 4096


def test_what_cannot_be_read_in_place_is_counted():
    m, k, n, g = 20_000, 1024, 1000, 4
    x, w, dy = m * k * 2, g * k * n * 2, m * n * 2
    for kw, room in ((dict(x=18), x), (dict(ldx=k + 1), x), (dict(w=24 + 2), w), (dict(ldw=n + 4), w), (dict(x=2, w=2), x + w)):
        assert room <= need(m, k, n, g, **kw) <= room + 4096 <= L().gc_grouped_linear_workspace_bytes(m, k, n, g, 0) + 4096, kw
    assert dy <= need(m, k, n, g, dx=1, dy=2) <= dy + 4096
    assert need(m, k, n, g, dx=1, x=2) <= 4096  # dX does not read X
    assert x <= need(m, k, n, g, dw=1, x=2) - need(m, k, n, g, dw=1) <= x + 4096
    assert need(m, k, n, g, dw=1, w=2) == need(m, k, n, g, dw=1)  # nor dW the weights
    assert m * 1024 * 2 <= need(m, 1021, n, g) <= m * 1024 * 2 + 4096  # a width of its own is a pitch of its own


def test_never_more_than_for_any_operands():
    for m, k, n, g in ((50, 24, 40, 3), (2708, 100, 47, 5), (5000, 999, 1001, 7), (300, 4096, 4096, 2)):
        for kw in (dict(), dict(x=2, w=2, dy=2), dict(ldx=k + 1, ldw=n + 1, lddy=n + 1)):
            assert 0 < need(m, k, n, g, **kw) <= L().gc_grouped_linear_workspace_bytes(m, k, n, g, 0)
            for dx, dw in ((1, 0), (0, 1), (1, 1)):
                assert 0 < need(m, k, n, g, dx, dw, **kw) <= L().gc_grouped_linear_workspace_bytes(m, k, n, g, 1)
    assert need(0, 8, 8, 1) == need(8, 0, 8, 1) == need(8, 8, 0, 1) == need(8, 8, 8, 0) == 0


def test_less_than_a_call_needs_is_refused():
    m, k, n, g = 20_000, 1024, 1000, 4

    def forward(x, room):
        return L().gc_grouped_linear_forward_bf16(x, k, 16, n, 16, m, k, n, g, 16, n, 16, room, None)

    def backward(dy, dx, dw, room):
        return L().gc_grouped_linear_backward_bf16(dy, n, 16, k, 16, n, 16, m, k, n, g, dx, k, dw, 16, room, None)

    assert forward(16, need(m, k, n, g) - 1) == -4 and forward(18, need(m, k, n, g, x=18) - 1) == -4
    assert backward(16, 16, None, need(m, k, n, g, dx=1) - 1) == -4
    assert backward(18, 16, None, need(m, k, n, g, dx=1, dy=18) - 1) == -4
    assert backward(16, 16, 16, need(m, k, n, g, dx=1, dw=1) - 1) == -4


@pytest.mark.gpu
def test_memory_of_a_call():
    """A product of large weights takes its result and little else; one whose rows lie on odd addresses a copy of them."""
    groups, m, k, n = 16, 4096, 2048, 2048
    w = torch.randn(groups, k, n, device="cuda").bfloat16()
    wide = torch.randn(m, k + 8, device="cuda").bfloat16()
    offsets = torch.linspace(0, m, groups + 1, device="cuda").int()
    row_bytes = m * k * 2
    for x, copies in ((wide[:, 8:], 0), (wide[:, 1:k + 1], 1)):
        want = torch.cat([x[int(a):int(b)].float() @ w[g].float() for g, (a, b) in enumerate(zip(offsets, offsets[1:]))])
        x, leaf = x.detach().requires_grad_(), w.detach()
        torch.cuda.synchronize()
        base = torch.cuda.memory_allocated()
        torch.cuda.reset_peak_memory_stats()
        y = gc.grouped_linear(x, leaf, offsets)
        (dx,) = torch.autograd.grad(y, x, torch.ones_like(y))
        peak = torch.cuda.max_memory_allocated() - base
        # y, its gradient and dx; room that is kept, up to 40 MB and a quarter; the weights are 134 MB
        assert peak <= 3 * row_bytes + copies * row_bytes + (50 << 20), peak
        assert float((y.float() - want).abs().max()) <= float(want.abs().max()) * 2.0 ** -7
