"""Calls for no sequence: nothing to do, and nothing to refuse."""
import ctypes

import rxmet_lib


def test_no_sequences_need_no_block_table():
    lib = rxmet_lib.load()
    buf = (ctypes.c_float * 16)()
    p = ctypes.addressof(buf) // 16 * 16
    cache = ctypes.byref(rxmet_lib.KvCache(p, p, p, p, 4, 2, 16, 64, 0))
    table = ctypes.byref(rxmet_lib.KvTable(None, 1, 0, 1))
    assert lib.rxmet_kv_append(cache, table, None, None, 0, 1, None, 128, 64, None, 128, 64, 0, None) == 0
    assert lib.rxmet_kv_read(cache, table, None, None, 0, 0, None, None, 0, None) == 0
    assert lib.rxmet_kv_attention(cache, table, None, None, 0, 1, 16, None, 128, 64, 2, 1.0, 1, 0, None, 1,
                                  None, None) == 0
    some = ctypes.byref(rxmet_lib.KvTable(None, 1, 1, 1))
    assert lib.rxmet_kv_append(cache, some, p, None, 1, 1, p, 128, 64, p, 128, 64, 0, None) == -22
    assert b"block table is empty" in lib.rxmet_last_error()
