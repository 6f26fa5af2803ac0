"""Limits of the cache's entry points that a launch's arithmetic has, refused on the CPU."""
import ctypes as C

from mako_b200 import _lib as c
from mako_b200 import lib
from tests.test_kv_arguments import AT, CACHE, SOME, fields, refused


def rows(**kw):
    good = dict(k=AT, v=AT, k_ld=128, v_ld=128, q=AT, q_out=AT, q_ld=256, q_out_ld=256, n_q_heads=4, type=1, n_tokens=5, positions=AT, slots=AT)
    return C.byref(fields(c.KvRowsC, **(good | kw)))


def test_query_heads_of_a_key_head_in_an_append():
    """65536 tokens of more would pass the 31 bits in which a block counts its rows."""
    cache = C.byref(fields(c.KvCacheC, **CACHE))
    for group in (8193, 20000, 1 << 20):
        refused(lib.mk_kv_append(SOME, cache, rows(n_q_heads=2 * group, q_ld=2 * group * 64, q_out_ld=2 * group * 64), None, None), "at most 8192")
    assert 65536 * (2 * 2 + 2 * 8192) < 2 ** 31 <= 65536 * (2 * 2 + 2 * 16384)
    assert lib.mk_kv_append(SOME, cache, rows(n_q_heads=2 * 8192, q_ld=2 * 8192 * 64, q_out_ld=2 * 8192 * 64, n_tokens=0), None, None) == 0
