"""What the cache's and the log-probabilities' entry points refuse, on the CPU: tensors of other devices, shapes and types in Python, sizes,
strides and alignments in the library, which looks at them before it touches the handle."""
import ctypes as C

import pytest
import torch

from mako_b200 import KvCache, MakoError, lib
from mako_b200 import _lib as c
from tests.test_round_ops_arguments import handle, on  # noqa: F401

H, B, I32 = torch.float16, torch.bfloat16, torch.int32


def logprobs(h):
    x = {"logits": on(3, 100), "tokens": on(3, 2, t=I32), "temperature": on(3), "mask": on(3, 4, t=I32)}
    return x, lambda: h.token_logprobs(**x, top=3)


def cache(x):
    return KvCache(x["k_codes"], x["v_codes"], x["k_scale"], x["v_scale"])


def pools():
    return {"k_codes": on(4, 2, 16, 64, t=torch.uint8), "v_codes": on(4, 2, 16, 64, t=torch.uint8), "k_scale": on(4, 2), "v_scale": on(4, 2)}


def append(h):
    x = pools() | {"k": on(5, 2, 64, t=B), "v": on(5, 2, 64, t=B), "slots": on(5, t=torch.int64), "q": on(5, 4, 64, t=B), "q_out": on(5, 4, 64, t=B),
                   "positions": on(5, t=I32), "inv_freq": on(32)}
    return x, lambda: h.kv_append(cache(x), **{k: x[k] for k in ("k", "v", "slots", "q", "q_out", "positions", "inv_freq")})


def attention(h):
    x = pools() | {"q": on(5, 4, 64, t=B), "block_table": on(3, 4, t=I32), "query_start": on(4, t=I32), "kv_len": on(3, t=I32), "out": on(5, 4, 64, t=B)}
    return x, lambda: h.kv_attention(x["q"], cache(x), x["block_table"], x["query_start"], x["kv_len"], out=x["out"])


CALLS = [logprobs, append, attention]


@pytest.mark.parametrize("call", CALLS)
def test_tensors_of_another_device_or_the_host_are_refused(handle, call):  # noqa: F811
    tensors, run = call(handle)
    with pytest.raises(MakoError, match="null argument"):
        run()
    for k, x in tensors.items():
        for where in (1, -1):
            x.where = where
            with pytest.raises(AssertionError):
                run()
                pytest.fail(k)
        x.where = 0


@pytest.mark.parametrize("call,name,other", [
    (logprobs, "tokens", on(3, 2, t=torch.int64)), (logprobs, "tokens", on(4, t=I32)), (logprobs, "temperature", on(4)),
    (logprobs, "temperature", on(3, t=torch.float64)), (logprobs, "mask", on(3, 3, t=I32)), (logprobs, "mask", on(2, 4, t=I32)),
    (logprobs, "logits", on(100, 3).t()), (append, "k", on(5, 2, 32, t=B)), (append, "k", on(5, 2, 64)), (append, "v", on(5, 2, 64, t=H)),
    (append, "v", on(5, 3, 64, t=B)), (append, "slots", on(5, t=I32)), (append, "slots", on(6, t=torch.int64)), (append, "q", on(5, 4, 64, t=H)),
    (append, "q_out", on(5, 2, 64, t=B)), (append, "q", on(4, 4, 64, t=B)), (append, "positions", on(5, t=torch.int64)),
    (append, "positions", on(4, t=I32)), (append, "inv_freq", on(32, t=torch.float64)), (append, "inv_freq", on(64)[::2]),
    (append, "k", on(5, 64, 2, t=B).transpose(1, 2)), (append, "k_codes", on(4, 2, 16, 64)), (append, "v_codes", on(4, 2, 8, 64, t=torch.uint8)),
    (append, "v_codes", on(4, 16, 2, 64, t=torch.uint8).transpose(1, 2)), (append, "k_scale", on(2, 4).t()), (append, "v_scale", on(4, 2, t=B)),
    (attention, "q", on(5, 4, 64)), (attention, "out", on(5, 4, 64, t=H)), (attention, "out", on(4, 4, 64, t=B)), (attention, "q", on(5, 4, 128, t=B)),
    (attention, "query_start", on(3, t=I32)), (attention, "kv_len", on(3, t=torch.int64)), (attention, "block_table", on(3, 4, t=torch.int64)),
    (attention, "block_table", on(4, 3, t=I32).t()), (attention, "k_codes", on(4, 2, 64, 16, t=torch.uint8).transpose(2, 3))])
def test_shapes_types_and_orders_are_refused(handle, call, name, other):  # noqa: F811
    tensors, run = call(handle)
    tensors[name] = other
    with pytest.raises((AssertionError, KeyError)):
        run()


def fields(struct, **kw):
    s = struct()
    for k, x in kw.items():
        setattr(s, k, x)
    return s


SOME = C.create_string_buffer(1 << 16)      # stands for a handle, which a refused call does not look at
AT = (C.addressof(SOME) + 255) & ~255        # and for device memory


def refused(rc, what):
    assert rc == c.MK_ERR_INVALID_ARGUMENT, rc
    assert what in lib.mk_last_error().decode(), lib.mk_last_error()


def test_the_library_refuses_rows_of_logits():
    good = dict(logits=AT, ld=100, type=0, rows=3, n_vocab=100, tokens=AT, n_given=2, n_top=3, temperature_all=1.0, mask=AT, mask_ld=4)
    out = [AT] * 5
    call = lambda **kw: lib.mk_token_logprobs(SOME, C.byref(fields(c.LogprobRowsC, **(good | kw))), *out, None)  # noqa: E731
    for kw, what in [(dict(type=3), "type"), (dict(n_vocab=0), "n_vocab"), (dict(n_vocab=1 << 29, ld=1 << 29, mask_ld=1 << 24), "n_vocab"),
                     (dict(n_top=65), "n_top"), (dict(ld=99), "ld"), (dict(mask_ld=3), "mask_ld"), (dict(temperature_all=float("nan")), "finite"),
                     (dict(temperature_all=float("inf")), "finite"), (dict(logits=None), "required"), (dict(tokens=None), "required"),
                     (dict(logits=AT + 2), "element"), (dict(logits=AT + 1, type=1), "element"), (dict(rows=(1 << 28) + 1), "rows")]:
        refused(call(**kw), what)
    assert call(rows=0) == 0
    refused(lib.mk_token_logprobs(None, None, *out, None), "null")


CACHE = dict(k=AT, v=AT, k_scale=AT, v_scale=AT, page_stride=2 * 16 * 64, head_stride=16 * 64, token_stride=64, n_pages=4, n_heads=2, page_size=16, dim=64)
BAD_CACHES = [(dict(page_size=(1 << 24) + 1), "page_size"), (dict(page_size=0), "page_size"), (dict(n_heads=0), "n_heads"), (dict(n_heads=65536), "n_heads"), (dict(dim=0), "dim"), (dict(dim=72), "dim"),
              (dict(dim=272, token_stride=272), "dim"), (dict(n_pages=1 << 31), "n_pages"), (dict(page_size=1 << 31), "page_size"),
              (dict(page_stride=8), "strides"), (dict(head_stride=1000), "strides"), (dict(token_stride=48), "strides"), (dict(token_stride=72), "strides"),
              (dict(k=None), "required"), (dict(v_scale=None), "required"), (dict(k=AT + 8), "16-byte"), (dict(v=AT + 4), "16-byte")]


def test_the_library_refuses_appends():
    rows = dict(k=AT, v=AT, k_ld=128, v_ld=128, q=AT, q_out=AT, q_ld=256, q_out_ld=256, n_q_heads=4, type=1, n_tokens=5, positions=AT, slots=AT)
    turn = dict(inv_freq=AT, dim=64, interleaved=0, scale=1.0)

    def call(of_cache={}, of_rows={}, of_turn={}):
        return lib.mk_kv_append(SOME, C.byref(fields(c.KvCacheC, **(CACHE | of_cache))), C.byref(fields(c.KvRowsC, **(rows | of_rows))),
                                C.byref(fields(c.RotaryC, **(turn | of_turn))), None)
    for kw, what in BAD_CACHES:
        refused(call(of_cache=kw), what)
    for kw, what in [(dict(type=0), "type"), (dict(k_ld=120), "k_ld"), (dict(v_ld=132), "v_ld"), (dict(q_out=None), "q_out"), (dict(n_q_heads=3), "n_q_heads"),
                     (dict(n_q_heads=0), "n_q_heads"), (dict(q_ld=248), "q_ld"), (dict(q_out_ld=260), "q_out_ld"), (dict(k=AT + 2), "16-byte"),
                     (dict(q=AT + 8), "16-byte"), (dict(q_out=AT + 8), "16-byte"), (dict(k=None), "required"), (dict(slots=None), "required"),
                     (dict(positions=None), "required"), (dict(n_tokens=1 << 31), "n_tokens")]:
        refused(call(of_rows=kw), what)
    for kw in (dict(dim=0), dict(dim=24), dict(dim=80), dict(scale=float("nan")), dict(scale=float("inf"))):
        refused(call(of_turn=kw), "rotation")
    assert call(of_rows=dict(n_tokens=0)) == 0
    refused(lib.mk_kv_append(SOME, None, None, None, None), "null")


def test_the_library_refuses_attention():
    rows = dict(q=AT, out=AT, q_ld=256, out_ld=256, n_q_heads=4, type=1, n_tokens=5, block_table=AT, table_ld=4, table_cols=4, query_start=AT, kv_len=AT, n_seq=3,
                max_new=2, scale=0.125, window=0, workspace=AT, workspace_bytes=1 << 40)

    def call(of_cache={}, **kw):
        return lib.mk_kv_attention(SOME, C.byref(fields(c.KvCacheC, **(CACHE | of_cache))), C.byref(fields(c.KvQueriesC, **(rows | kw))), None)
    for kw, what in BAD_CACHES + [(dict(dim=48), "neither 64 nor 128")]:
        refused(call(kw), what)
    for kw, what in [(dict(type=0), "type"), (dict(n_q_heads=0), "n_q_heads"), (dict(n_q_heads=5), "n_q_heads"), (dict(q_ld=250), "q_ld"), (dict(out_ld=260), "out_ld"),
                     (dict(n_seq=8193), "n_seq"), (dict(table_ld=3), "table_ld"), (dict(table_cols=1 << 31, table_ld=1 << 31), "table_cols"),
                     (dict(scale=float("nan")), "scale"), (dict(window=1 << 31), "window"), (dict(q=AT + 8), "16-byte"), (dict(out=AT + 2), "16-byte"),
                     (dict(workspace=AT + 8), "16-byte"), (dict(q=None), "required"), (dict(block_table=None), "required"), (dict(kv_len=None), "required"),
                     (dict(workspace=None), "workspace"), (dict(workspace_bytes=1000), "workspace"), (dict(n_tokens=(1 << 30) + 1), "n_tokens")]:
        refused(call(**kw), what)
    assert call(n_seq=0) == 0 and call(n_tokens=0) == 0
    refused(call(), "out is q")
    refused(lib.mk_kv_attention(None, None, None, None), "null")
