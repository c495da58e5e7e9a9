"""The entry points of the grouped product answer bad arguments without touching a GPU."""
import pytest
import torch

import graphcuda_b200 as gc
from graphcuda_b200 import _lib

M, K, N, G = 50, 24, 40, 3
L = _lib.lib


def _forward(x=16, ldx=K, w=16, ldw=N, off=16, m=M, k=K, n=N, g=G, y=16, ldy=N, ws=16, wsb=None):
    need = L().gc_grouped_linear_workspace_bytes(M, K, N, G, 0)
    return L().gc_grouped_linear_forward_bf16(x, ldx, w, ldw, off, m, k, n, g, y, ldy, ws, need if wsb is None else wsb, None)


def _backward(dy=16, lddy=N, x=16, ldx=K, w=16, ldw=N, off=16, m=M, k=K, n=N, g=G, dx=16, lddx=K, dw=16, ws=16, wsb=None):
    need = L().gc_grouped_linear_workspace_bytes(M, K, N, G, 1)
    return L().gc_grouped_linear_backward_bf16(dy, lddy, x, ldx, w, ldw, off, m, k, n, g, dx, lddx, dw, ws, need if wsb is None else wsb, None)


@pytest.mark.parametrize("call", [_forward, _backward])
def test_what_both_refuse(call):
    for bad in (dict(m=-1), dict(k=-1), dict(n=-1), dict(g=-1), dict(ldx=K - 1), dict(ldw=N - 1), dict(off=None), dict(x=None), dict(w=None),
                dict(ws=24)):
        assert call(**bad) == -1, bad
    assert call(m=1 << 31) == -2 and call(g=(1 << 20) + 1) == -2
    assert call(ws=None) == -4 and call(wsb=L().gc_grouped_linear_workspace_bytes(M, K, N, G, int(call is _backward)) - 1) == -4


def test_forward_arguments():
    assert _forward(ldy=N - 1) == -1 and _forward(y=None) == -1
    assert _forward(m=0, x=None, y=None) == 0 and _forward(n=0, ldw=0, ldy=0, y=None) == 0


def test_backward_arguments():
    assert _backward(lddy=N - 1) == -1 and _backward(lddx=K - 1) == -1 and _backward(dy=None) == -1
    assert _backward(dx=None, dw=None, lddx=0, ws=None, wsb=0) == 0
    assert _backward(m=0, dx=None, dw=None, ws=None, wsb=0) == 0


def test_queries():
    q = L().gc_grouped_linear_workspace_bytes
    for back in (0, 1):
        assert q(0, K, N, G, back) == q(M, 0, N, G, back) == q(M, K, 0, G, back) == q(M, K, N, 0, back) == q(-1, K, N, G, back) == 0
        assert 0 < q(M, K, N, G, back) <= q(M + 1000, K, N, G + 1, back)


def test_cpu_tensors_are_refused():
    with pytest.raises(RuntimeError, match="CUDA"):
        gc.grouped_linear(torch.zeros(4, 8, dtype=torch.bfloat16), torch.zeros(2, 8, 8, dtype=torch.bfloat16),
                          torch.tensor([0, 1, 4], dtype=torch.int32))


def test_module():
    torch.manual_seed(0)
    layer = gc.GroupedLinear(16, 24, 3)
    assert layer.weight.shape == (3, 16, 24) and layer.weight.dtype == torch.bfloat16 and set(layer.state_dict()) == {"weight"}
