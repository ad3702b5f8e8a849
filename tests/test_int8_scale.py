"""int8 attention: scales whose product with log2(e) is no 32-bit number are refused
(CPU)."""
import ctypes as C
import importlib

L = importlib.import_module("truellm-engine_b200._lib")
P = 1 << 20  # an aligned address that no refused call touches


def test_a_scale_that_overflows_is_refused():
    lib = L.lib()
    cache = L.TkvInt8Cache(pool=P, num_pages=4, n_kv_heads=2, head_dim=128)

    def call(scale):  # no tokens: an accepted call launches nothing
        return lib.tkv_int8_attend(C.byref(cache), P, L.TKV_BF16, (C.c_int64 * 2)(1024, 128), P,
                                   L.TKV_BF16, P, P, 4, P, 2, 8, 0, 4, 64, 0, scale, P, 1 << 30,
                                   None, None)
    assert call(2.3e38) == call(1e-45) == L.TKV_OK
    assert call(2.4e38) == call(3.4e38) == L.TKV_INVALID_ARGUMENT
