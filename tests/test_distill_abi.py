"""The entry points of the distillation loss answer bad arguments without touching a GPU."""
import pytest
import torch

import graphcuda_b200 as gc
from graphcuda_b200 import _lib

M, C, K = 5, 9, 3
L = _lib.lib


def _forward(z=16, zt=0, ldz=C, t=16, tt=0, ldt=K, i=16, bits=64, ldi=K, mask=None, m=M, c=C, k=K, temp=1.0, scale=1.0, loss=16,
             stats=16, dz=None, lddz=C, pad=0, ws=16, wsb=None):
    return L().gc_distill_forward(z, zt, ldz, t, tt, ldt, i, bits, ldi, mask, m, c, k, temp, scale, loss, stats, dz, lddz, pad, ws,
                                  L().gc_distill_workspace_bytes(M, C) if wsb is None else wsb, None)


def _backward(z=16, zt=0, ldz=C, t=16, tt=0, ldt=K, i=16, bits=64, ldi=K, stats=16, m=M, c=C, k=K, temp=1.0, scale=1.0, g=16, dz=16,
              lddz=C, pad=0, made=0):
    return L().gc_distill_backward(z, zt, ldz, t, tt, ldt, i, bits, ldi, stats, m, c, k, temp, scale, g, dz, lddz, pad, made, None)


@pytest.mark.parametrize("call", [_forward, _backward])
def test_what_both_refuse(call):
    for bad in (dict(m=-1), dict(c=0), dict(k=-1), dict(zt=2), dict(tt=3), dict(bits=16), dict(ldz=C - 1), dict(ldt=K - 1),
                dict(ldi=K - 1), dict(temp=0.0), dict(temp=-1.0), dict(temp=float("inf")), dict(temp=float("nan")), dict(temp=1e-39),
                dict(z=None), dict(t=None), dict(i=None), dict(stats=None), dict(stats=8)):
        assert call(**bad) == -1, bad
    assert call(k=1025, ldt=1025, ldi=1025) == -2 and b"1024" in L().gc_last_error()
    assert call(c=1 << 31, ldz=1 << 31, **({"lddz": 1 << 31} if call is _backward else {})) == -2


def test_forward_arguments():
    assert _forward(loss=None) == -1
    assert _forward(dz=16, lddz=C - 1) == -1 and _forward(dz=16, pad=8, lddz=C + 8) == -1
    assert _forward(dz=16, c=5000, ldz=5000, lddz=5000) == -1 and b"rows like these" in L().gc_last_error()
    assert _forward(ws=None) == -4 and _forward(wsb=L().gc_distill_workspace_bytes(M, C) - 1) == -4 and _forward(ws=24) == -1
    assert L().gc_distill_workspace_bytes(-1, C) == L().gc_distill_workspace_bytes(M, 0) == 0
    assert L().gc_distill_workspace_bytes(4, 100_000) > L().gc_distill_workspace_bytes(4, 100)


def test_backward_arguments():
    assert _backward(g=None) == -1 and _backward(dz=None) == -1 and _backward(lddz=C - 1) == -1
    assert _backward(pad=-1) == -1 and _backward(pad=8, lddz=C + 8) == -1 and _backward(pad=2, lddz=C + 1) == -1
    assert _backward(m=0, z=None, t=None, i=None, stats=None, dz=None, g=None) == 0


def test_which_rows_go_in_one_pass():
    def one(z, t, ldz, lddz, m, c, k=8):
        return L().gc_distill_one_pass(z, t, ldz, lddz, m, c, k)

    assert one(16, 0, 8192, 8192, 1000, 8192) and one(16, 1, 90_001, 90_001, 1000, 90_001)
    assert one(16, 0, 47, 47, 100_000, 47) and one(20, 0, 4099, 4096, 3, 4096, 1024)  # short rows, wherever they lie
    assert not one(16, 1, 4097, 4097, 10_000, 4097, 300)  # neither short nor with a short list
    assert not one(16, 0, 50_689, 50_689, 1000, 50_689) and not one(16, 1, 101_377, 101_377, 1000, 101_377)  # longer than the ring
    assert not one(16, 0, 8192, 8192, 100, 8192)     # few rows
    assert not one(20, 0, 8192, 8192, 1000, 8192) and not one(16, 0, 8193, 8192, 1000, 8192)  # the rows lie differently
    assert not one(16, 2, 8192, 8192, 1000, 8192) and not one(16, 0, 8192, 8192, 1000, 8192, 257)


def test_cpu_tensors_are_refused():
    with pytest.raises(RuntimeError, match="CUDA"):
        gc.distill_loss(torch.zeros(2, 4), torch.zeros(2, 1), torch.zeros(2, 1, dtype=torch.int64))
