"""The types that gc_adamw_step takes, without touching a GPU."""
import ctypes as C

from graphcuda_b200 import _lib

FOLLOW = 256


def test_only_parameters_beside_masters_are_followed():
    L = _lib.lib()
    one, size = (C.c_void_p * 1)(16), (C.c_int64 * 1)(5)

    def call(kind, master=one):
        return L.gc_adamw_step(1, one, kind, one, master, one, one, None, None, size, 32, 0.1, 0.9, 0.99, 1e-8, 0.0, 0, None, None)

    assert call(_lib.TYPE_BF16 | FOLLOW) == -1 and b"null state" in L.gc_last_error()
    null = (C.c_void_p * 1)(None)
    for kind in (_lib.TYPE_F32 | FOLLOW, _lib.TYPE_E4M3 | FOLLOW, _lib.TYPE_BF16 | 512, _lib.TYPE_BF16 | -256, 3):
        assert L.gc_adamw_step(1, one, kind, one, one, one, one, None, None, size, 32, 0.1, 0.9, 0.99, 1e-8, 0.0, 0, 16, None) == -1
        assert b"followed" in L.gc_last_error()
    assert L.gc_adamw_step(1, one, _lib.TYPE_BF16 | FOLLOW, one, null, one, one, None, None, size, 32, 0.1, 0.9, 0.99, 1e-8, 0.0, 0, 16,
                           None) == -1 and b"tensor 0" in L.gc_last_error()
    assert L.gc_adamw_step(1, one, _lib.TYPE_BF16 | FOLLOW, one, None, one, one, None, None, size, 32, 0.1, 0.9, 0.99, 1e-8, 0.0, 0, 16,
                           None) == -1 and b"masters" in L.gc_last_error()
