"""The expanded attention's largest launches (CPU only): 2^24 blocks of 256 threads are one too many."""

import ctypes

from mla_kv_quant_amd import _lib

P = ctypes.c_void_p(4096)


def test_two_to_the_24_blocks_are_refused():
    lib = _lib.load()

    def call(T, B, H):
        rc = lib.rolaq_expanded_attend_fwd(P, H * 192, 192, P, H * 256, 256, P, 64, P, P, T, 50, B, H, 128, 64, 128, 1, 0.1, 1,
                                           P, H * 128, 128, None, None, 0, None)
        return rc, lib.rolaq_last_error().decode()

    for T, B, H in ((5, 1 << 17, 128), (31, 1 << 18, 64), (5, (1 << 17) + 1, 128)):
        rc, text = call(T, B, H)
        assert rc == _lib.ROLAQ_ERR_INVALID and "too large" in text, (rc, text)
