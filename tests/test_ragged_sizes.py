"""Sizes whose products pass 63 bits are refused at the C entries of the ragged cache, before anything is worked out from a product that has wrapped
round (to a number of pages that is 0, for one).  The addresses are made up; nothing reads them."""
import ctypes as C

import pytest

UNSUPPORTED = -4
I32_MAX = 2 ** 31 - 1


def store(base, layers=1, obs=1, n_kv=1, hd=64, cap=8):
    from vla_cpp_b200 import api

    return api._KvStoreC(base, base + (1 << 40), layers, obs, n_kv, hd, cap, 0)


PAGES = [(2 ** 22, 2 ** 21, 2 ** 21), (2 ** 30, 2 ** 30, 16), (2 ** 16, 2 ** 16, 2 ** 31 - 1), (I32_MAX,) * 3]  # layers, observations, kv heads


@pytest.mark.parametrize("layers,obs,n_kv", PAGES)
def test_more_pages_than_there_can_be(layers, obs, n_kv):
    from vla_cpp_b200 import api

    L = api.lib()
    st, dst = (store(b << 45, layers, obs, n_kv) for b in (1, 2))
    p = [C.c_void_p((8 + i) << 45) for i in range(6)]
    assert L.vlab200_kv_evict(C.byref(st), C.byref(dst), p[0], None, 8, 4, 0, 0, p[1], None, None, None) == UNSUPPORTED
    assert L.vlab200_cross_attention(C.byref(st), 0, p[0], p[1], p[2], 1, n_kv, None, 8, None, 0.0, None, 0, None) == UNSUPPORTED
    assert L.vlab200_cross_attention_ws_bytes(C.byref(st), 1, n_kv, 8) == -1
    assert L.vlab200_key_mass(C.byref(st), 0, p[0], p[1], None, p[2], 1, n_kv, None, 8, None, 0.0, 1.0, None) == UNSUPPORTED


def test_more_blocks_of_scores_than_are_counted():
    from vla_cpp_b200 import api

    L = api.lib()
    p = [C.c_void_p((8 + i) << 45) for i in range(6)]
    st = store(1 << 45, 1, 2 ** 30, 1, cap=I32_MAX)  # 2^30 items x 2^23 units x 2^24 blocks
    assert L.vlab200_cross_attention(C.byref(st), 0, p[0], p[1], p[2], 2 ** 30, 1, None, I32_MAX, None, 0.0, None, 0, None) == UNSUPPORTED
    assert L.vlab200_cross_attention_ws_bytes(C.byref(st), 2 ** 30, 1, I32_MAX) == -1
    assert L.vlab200_key_mass(C.byref(st), 0, p[0], p[1], None, p[2], 2 ** 30, 1, None, I32_MAX, None, 0.0, 1.0, None) == UNSUPPORTED


@pytest.mark.parametrize("layers,obs,S,n_q,n_kv,stride", [
    (1, 1, 1, I32_MAX, 1, 2 ** 40),              # heads of a row: 2^31 + 1
    (1, 1, 1, 1, 2 ** 30, 2 ** 40),
    (1, 2 ** 20, 2 ** 20, 1, 1, 2 ** 40),        # rows x stride
    (2 ** 30, 2 ** 25, 1, 1, 1024, 2 ** 40),     # pages
])
def test_rotation_of_more_than_there_can_be(layers, obs, S, n_q, n_kv, stride):
    from vla_cpp_b200 import api

    st = store(1 << 45, layers, obs, n_kv)
    a = api._QkNormRopeArgs((8 << 45), stride, None, None, None, None, None, None, (9 << 45), S, n_q, 0, 0, 0, 1, 1e-6, 1.0)
    assert api.lib().vlab200_qk_norm_rope_append(C.byref(st), 0, C.byref(a), None) == UNSUPPORTED
