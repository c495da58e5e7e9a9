"""The entry points of the norm and of AdamW answer bad arguments without touching a GPU."""
from graphcuda_b200 import _lib

F32, BF16, E4M3 = _lib.TYPE_F32, _lib.TYPE_BF16, _lib.TYPE_E4M3


def _forward(x=16, xt=F32, r=16, st=F32, M=4, N=8, y=16, yt=F32, scale=None, ld=8, w=16):
    return _lib.lib().gc_rms_norm_forward(x, xt, ld, r, ld, st, w, M, N, 1e-6, y, yt, ld, 16, ld, None, scale, None)


def test_norm_arguments():
    L = _lib.lib()
    assert _forward(M=-1) == -1 and b"negative" in L.gc_last_error()
    assert _forward(xt=E4M3) == -1 and _forward(yt=7) == -1
    assert _forward(xt=F32, st=BF16) == -1  # an fp32 x beside a bf16 stream
    assert _forward(xt=BF16, st=F32, r=None) == -1  # without a residual the stream is x
    assert _forward(x=None) == -1 and _forward(w=None) == -1 and _forward(y=None) == -1
    assert _forward(yt=E4M3) == -1 and b"scales" in L.gc_last_error()
    assert _forward(ld=7) == -1 and b"leading dimension" in L.gc_last_error()
    assert _forward(N=1 << 31, ld=1 << 31) == -1
    assert _forward(M=0, x=None) == 0 and _forward(N=0) == 0


def _backward(M=1000, N=8, dy=16, yt=F32, h=16, r=None, st=F32, dx=16, xt=F32, dres=None, dw=16, ws=None, wsb=0, ld=8):
    return _lib.lib().gc_rms_norm_backward(dy, yt, ld, None, ld, h, ld, r, ld, st, 16, 16, M, N, dx, xt, ld, dres, ld, dw,
                                           ws, wsb, None)


def test_norm_backward_arguments():
    L = _lib.lib()
    need = L.gc_rms_norm_backward_workspace_bytes(1000, 8)
    assert need % 32 == 0 and need > 0  # whole partial rows
    assert L.gc_rms_norm_backward_workspace_bytes(1, 8) == 0 and L.gc_rms_norm_backward_workspace_bytes(0, 8) == 0
    assert _backward() == -4  # several CTAs and no room for their sums
    assert _backward(ws=16, wsb=need - 4) == -4
    assert _backward(ws=18, wsb=need) == -1
    assert _backward(r=16) == -1 and b"exact" in L.gc_last_error()
    assert _backward(dx=None, dres=16) == -1
    assert _backward(dy=None) == -1 and _backward(h=None) == -1 and _backward(ld=7) == -1
    assert _backward(yt=E4M3) == -1
    assert _backward(dx=None, dw=None) == 0  # nothing wanted


def test_adamw_arguments():
    import ctypes as C
    L = _lib.lib()
    one, size = (C.c_void_p * 1)(16), (C.c_int64 * 1)(5)
    null = (C.c_void_p * 1)(None)

    def call(n=1, p=one, kind=F32, g=one, master=None, m=one, v=one, ms=None, vs=None, n_el=size, bits=32, state=16):
        return L.gc_adamw_step(n, p, kind, g, master, m, v, ms, vs, n_el, bits, 0.1, 0.9, 0.99, 1e-8, 0.0, 0, state, None)

    assert call(state=None) == -1 and call(n=-1) == -1 and call(kind=E4M3) == -1 and call(bits=16) == -1
    assert call(p=None) == -1 and call(g=null) == -1 and b"tensor 0" in L.gc_last_error()
    assert call(kind=BF16) == -1 and b"masters" in L.gc_last_error()
    assert call(kind=BF16, master=null) == -1
    assert call(bits=8) == -1 and b"scales" in L.gc_last_error()
    assert call(bits=8, ms=one, vs=null) == -1
    assert call(n_el=(C.c_int64 * 1)(-1)) == -1
    assert L.gc_adamw_moments_f32(1, one, one, one, null, size, one, one, None) == -1
    assert L.gc_adamw_moments_f32(-1, None, None, None, None, None, None, None, None) == -1
    assert L.gc_adamw_moments_f32(0, None, None, None, None, None, None, None, None) == 0
