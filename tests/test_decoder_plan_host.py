"""How attention calls are cut into launches, seen from the host: the workspace that they ask for."""
import ctypes

import rxmet_lib


def workspace(heads, dim, seqs, queries, q_heads, max_query, max_length, window=0):
    cache = rxmet_lib.KvCache(None, None, None, None, 1, heads, 64, dim, 0)
    return rxmet_lib.load().rxmet_kv_attention_workspace_bytes(ctypes.byref(cache), seqs, queries, q_heads,
                                                               max_query, max_length, window)


def test_a_long_axis_is_split_where_rows_are_few():
    assert workspace(8, 128, 2, 2, 32, 1, 32768) > 0
    assert workspace(8, 128, 64, 64, 64, 1, 512) == 0


def test_rows_beyond_a_launch_of_the_join_are_not_split():
    """2^24 rows of which max_query says 1: a workgroup of the join for each would be 2^32 threads."""
    assert workspace(8, 64, 1, 1 << 18, 64, 1, 1 << 17) == 0
    assert workspace(8, 64, 1, (1 << 18) - 1, 64, 1, 1 << 17) > 0
