"""CPU: sizes at which the kernels' 32-bit counts would overflow are refused before any launch."""

import ctypes as C

from utttcompanion_b200 import _lib

SIZE = _lib.UTTT_ERR_UNSUPPORTED


def _buf():
    b = C.create_string_buffer(4096)
    return b, (C.addressof(b) + 255) // 256 * 256


def test_fork_counts_a_heads_pieces_in_an_int():
    lib = _lib.load()
    keep, p = _buf()
    one, two = (C.c_int * 1)(0), (C.c_int * 1)(1)
    for hd, W in ((8, 2 ** 31 - 1), (8, 2 ** 30 + 1), (128, 2 ** 26 + 1)):
        st = lib.uttt_kv_ring_fork(1, 1, 1, hd, W, 2, p, p, 2 * W * hd, one, two, None, None)
        assert st == SIZE, (hd, W)
    assert lib.uttt_kv_ring_fork(1, 1, 1, 8, 1, 2 ** 30 + 1, p, p, 2 ** 34, one, two, None, None) == SIZE


def test_commit_counts_a_rows_pieces_in_an_int():
    lib = _lib.load()
    keep, p = _buf()
    n_kv, hd = 1 << 16, 1 << 16
    stride = 64 * n_kv * hd
    assert lib.uttt_kv_ring_commit(1, 1, 64, n_kv, hd, 1, 1, p, p, stride, p, p, stride, p, p, p, p, None) == SIZE


def test_tree_attention_tells_places_by_ints():
    lib = _lib.load()
    keep, p = _buf()
    for W in (2 ** 30 + 1, 2 ** 31 - 1):
        assert lib.uttt_attn_tree(1, 4, 4, 2, 64, W, 1, 16, p, 512, p, None, p, p, p, p, p, p, p, p, p, 256,
                                  None) == SIZE
