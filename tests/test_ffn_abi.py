"""The entry points of the gated block answer bad arguments without touching a GPU."""
import ctypes as C

import pytest

from graphcuda_b200 import _lib

M, D, H, O = 9, 8, 24, 16
L = _lib.lib
NEED = dict(fwd=lambda: L().gc_gated_ffn_workspace_bytes(M, D, H, O, 0), bwd=lambda: L().gc_gated_ffn_workspace_bytes(M, D, H, O, 1),
            f8=lambda: L().gc_gated_ffn_e4m3_workspace_bytes(M, D, H, O))


def _forward(x=16, ldx=D, wi=16, ldwi=2 * H, wo=16, ldwo=O, m=M, d=D, h=H, o=O, act=0, y=16, ldy=O, saved=None, ws=16, wsb=None):
    return L().gc_gated_ffn_forward_bf16(x, ldx, wi, ldwi, wo, ldwo, m, d, h, o, act, y, ldy, saved, ws,
                                         NEED["fwd"]() if wsb is None else wsb, None)


def _backward(dy=16, lddy=O, x=16, ldx=D, wi=16, ldwi=2 * H, wo=16, ldwo=O, saved=16, m=M, d=D, h=H, o=O, act=0, dx=16, lddx=D,
              dwi=16, lddwi=2 * H, dwo=16, lddwo=O, ws=16, wsb=None):
    return L().gc_gated_ffn_backward_bf16(dy, lddy, x, ldx, wi, ldwi, wo, ldwo, saved, m, d, h, o, act, dx, lddx, dwi, lddwi,
                                          dwo, lddwo, ws, NEED["bwd"]() if wsb is None else wsb, None)


def _eight(x=16, ldx=D, xs=16, w=16, ldw=D, wscale=16, wo=16, ldwo=O, m=M, d=D, h=H, o=O, act=0, y=16, ldy=O, ws=16, wsb=None):
    f = C.POINTER(C.c_float)
    return L().gc_gated_ffn_forward_e4m3(x, ldx, C.cast(xs, f) if xs else None, w, ldw, C.cast(wscale, f) if wscale else None, wo, ldwo,
                                         m, d, h, o, act, y, ldy, ws, NEED["f8"]() if wsb is None else wsb, None)


@pytest.mark.parametrize("call,need", [(_forward, "fwd"), (_backward, "bwd"), (_eight, "f8")])
def test_what_all_refuse(call, need):
    for size in "mdho":
        assert call(**{size: -1}) == -1 and b"negative" in L().gc_last_error()
    assert call(act=3) == -1 and call(act=-1) == -1 and b"activation" in L().gc_last_error()
    assert call(ldx=D - 1) == -1 and b"leading dimension" in L().gc_last_error()
    assert call(ldwo=O - 1) == -1 and call(wo=None) == -1 and call(x=None) == -1
    big = 1 << 31
    assert call(m=big) == -2  # beyond 32-bit coordinates: unsupported, not a bad argument
    assert call(ws=None) == -4 and call(wsb=NEED[need]() - 1) == -4 and b"workspace" in L().gc_last_error()
    assert call(ws=24) == -1 and b"aligned" in L().gc_last_error()


def test_forward_arguments():
    assert _forward(ldwi=2 * H - 1) == -1 and _forward(ldy=O - 1) == -1
    assert _forward(wi=None) == -1 and _forward(y=None) == -1
    assert _forward(saved=24) == -1 and b"saved" in L().gc_last_error()
    assert _forward(m=0, x=None, y=None) == 0 and _forward(o=0, ldwo=0, ldy=0, y=None) == 0
    assert L().gc_gated_ffn_saved_bytes(0, H) == 0 and L().gc_gated_ffn_saved_bytes(M, 0) == 0
    assert L().gc_gated_ffn_saved_bytes(M, H) >= 6 * M * H


def test_backward_arguments():
    assert _backward(lddy=O - 1) == -1 and _backward(lddx=D - 1) == -1 and _backward(lddwi=2 * H - 1) == -1
    assert _backward(lddwo=O - 1) == -1 and _backward(ldwi=2 * H - 1) == -1
    assert _backward(dy=None) == -1 and _backward(wi=None) == -1 and _backward(saved=None) == -1 and _backward(saved=8) == -1
    assert _backward(dx=None, dwi=None, dwo=None, lddx=0, lddwi=0, lddwo=0, ws=None, wsb=0) == 0  # nothing wanted
    assert _backward(m=0, dx=None, dwi=None, dwo=None, ws=None, wsb=0) == 0


def test_eight_bit_arguments():
    assert _eight(ldw=D - 1) == -1 and _eight(ldy=O - 1) == -1
    assert _eight(m=0, x=None, y=None) == 0
    assert _eight(xs=None) == -1 and _eight(wscale=None) == -1 and _eight(w=None) == -1 and _eight(y=None) == -1


@pytest.mark.parametrize("query", [lambda *s: L().gc_gated_ffn_workspace_bytes(*s, 0), lambda *s: L().gc_gated_ffn_workspace_bytes(*s, 1),
                                   lambda *s: L().gc_gated_ffn_e4m3_workspace_bytes(*s)])
def test_queries(query):
    assert query(0, D, H, O) == query(M, 0, H, O) == query(M, D, H, 0) == query(-1, D, H, O) == 0
    assert query(1 << 31, D, H, O) == 0
    assert 0 < query(M, D, H, O) <= query(M + 128, D, H, O)
