"""Argument checks of the clip entry point that takes its limit in 64 bits; nothing is launched."""
import ctypes
import math


def test_refusals():
    from protein_lig_sedd_amd import _lib
    L = _lib.lib()
    buf = ctypes.create_string_buffer(128)
    p = (ctypes.addressof(buf) + 63) // 64 * 64
    table = ((ctypes.c_void_p * 1)(p), (ctypes.c_int64 * 1)(4), (ctypes.c_int32 * 1)(0), 1)

    def call(limit, ws=p, doubles=5000, out=p):
        num = None if limit is None else ctypes.byref(ctypes.c_double(limit))
        return L.sedd_multi_norm_clip_f64(*table, num, ws, doubles, out, None)

    for args in ((None,), (-1.0,), (-1e-300,), (math.nan,), (1.0, None), (1.0, p, 4096), (1.0, p, 5000, None)):
        assert call(*args) == -1, args
        assert b"multi_norm_clip" in L.sedd_last_error()
