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


def test_outputs_that_overlap_what_is_read():
    """By a row, by a part of one, from in front and from behind, with strides that differ; outputs beside their inputs in the same rows are taken."""
    cache = C.byref(fields(c.KvCacheC, **CACHE))  # 2 heads of 64
    base = AT + 4096
    q = dict(q=base, q_ld=512, n_q_heads=4, k=base + 2 * 256, v=base + 2 * 384, k_ld=512, v_ld=512)  # one projection: q, k, v side by side

    def append(out, ld=512, **kw):
        return lib.mk_kv_append(SOME, cache, rows(**(q | dict(q_out=out, q_out_ld=ld) | kw)), None, None)

    for out, ld in [(base + 16, 512), (base - 16, 512), (base + 2 * 512, 512), (base + 2 * 248, 512), (base + 2 * 256, 512), (base + 2 * 384, 512),
                    (base, 256), (base, 520), (base + 2 * 4 * 512, 512), (base - 2 * 4 * 512, 512), (base - 2 * 4 * 512 - 2 * 248, 512),
                    (base + 2 * 4 * 512 + 2 * 504, 512), (base - 2 * 2048, 256 + 264)]:
        refused(append(out, ld), "q_out overlaps")

    def attend(out, ld=512, **kw):
        good = dict(q=base, out=out, q_ld=512, out_ld=ld, n_q_heads=4, type=1, n_tokens=5, block_table=AT, table_ld=4, table_cols=4, query_start=AT, kv_len=AT, n_seq=3,
                    max_new=2, scale=0.125, window=0, workspace=AT, workspace_bytes=1 << 40)
        return lib.mk_kv_attention(SOME, cache, C.byref(fields(c.KvQueriesC, **(good | kw))), None)
    for out, ld in [(base, 512), (base + 16, 512), (base - 16, 512), (base + 2 * 248, 512), (base - 2 * 248, 512), (base + 2 * 512, 512), (base, 256), (base + 2 * 256, 264),
                    (base + 2 * 4 * 512 + 2 * 248, 512), (base - 2 * 4 * 512, 512)]:
        refused(attend(out, ld), "out is q")
