"""Attention where a block table has fewer columns than a sequence has pages: the keys behind them are not there, and positions are those of the
whole length."""
import math

import numpy as np
import pytest
import torch

from tests import kv_oracle as oracle
from tests.test_gpu_kv_attention import make, sampler  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("new", [1, 5, 40, 150])
@pytest.mark.parametrize("page", [16, 24])
@pytest.mark.parametrize("columns", [0, 1, 9])
@pytest.mark.parametrize("window", [0, 30, 170])
def test_keys_behind_the_table_are_not_there(sampler, new, page, columns, window):  # noqa: F811
    rng = np.random.default_rng(new + page + columns)
    cache, q, table, start, kv_len = make(rng, [300, 170, 250], [new, new, 1], 2, 8, 64, page, "bf16")
    none = table.copy()
    none[:, columns:] = -1  # the same keys, by a table that has all columns
    cuda = lambda x: torch.from_numpy(x).cuda()  # noqa: E731
    out = torch.full_like(q, 7.0)
    sampler.kv_attention(q, cache, cuda(table)[:, :columns], cuda(start), cuda(kv_len), max_new=new, window=window, out=out)
    wide = lambda x, s: x.float().cpu().double() * s.double().cpu().view(*s.shape, 1, 1)  # noqa: E731
    want, bound = oracle.attention(q.double().cpu(), wide(cache.k, cache.k_scale), wide(cache.v, cache.v_scale), none, start, kv_len, page,
                                   1 / math.sqrt(64), window, q.dtype)
    got = out.double().cpu()
    for t in want:
        assert ((got[t] - want[t]).abs() <= bound[t]).all(), t
    assert (got[int(start[-1]):] == 7.0).all()


def test_lengths_beyond_all_pages(sampler):  # noqa: F811
    """The longest length there is, of a sequence whose keys behind the table are all that its window reaches."""
    rng = np.random.default_rng(1)
    cache, q, table, start, kv_len = make(rng, [300, 40], [70, 3], 1, 4, 128, 16, "fp16")
    cuda = lambda x: torch.from_numpy(x).cuda()  # noqa: E731
    kv_len[:] = 2 ** 31 - 1
    out = sampler.kv_attention(q, cache, cuda(table), cuda(start), cuda(kv_len), max_new=70, window=1000, out=torch.full_like(q, 7.0))
    assert (out[:73] == 0).all() and (out[73:] == 7).all()
    # without a window every key that is there is seen, by each token alike
    for x in (cache.k, cache.v):
        raw = x.view(torch.uint8)
        raw[(raw & 0x7f) == 0x7f] = 0x30
    out = sampler.kv_attention(q, cache, cuda(table), cuda(start), cuda(kv_len), max_new=70).double().cpu()
    wide = lambda x, s: x.float().cpu().double() * s.double().cpu().view(*s.shape, 1, 1)  # noqa: E731
    k, v = wide(cache.k, cache.k_scale), wide(cache.v, cache.v_scale)
    for t, of in ((0, 0), (69, 0), (71, 1)):
        held = int((table[of] >= 0).sum()) * 16
        want, bound = oracle.attention(q[t:t + 1].double().cpu(), k, v, table[of:of + 1], [0, 1], [held], 16, 1 / math.sqrt(128), 0, q.dtype)
        assert ((out[t] - want[0]).abs() <= bound[0]).all(), t


@pytest.mark.parametrize("new", [1, 90])
def test_a_cache_without_pages(sampler, new):  # noqa: F811
    """Whatever the table says, no page is there: zeros."""
    from mako_b200 import KvCache
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    for page, dim in ((16, 128), (24, 64)):
        q = torch.randn(new + 2, 4, dim, device="cuda").half()
        out = sampler.kv_attention(q, KvCache.empty(0, 2, page, dim), i32(0, 1, 2, 3, -1, 5).view(1, 6), i32(0, new), i32(90), max_new=new, out=torch.full_like(q, 7.0))
        assert (out[:new] == 0).all() and (out[new:] == 7).all()
        k = torch.randn(3, 2, dim, device="cuda").half()
        sampler.kv_append(KvCache.empty(0, 2, page, dim), k, k.clone(), torch.tensor([-1, 0, 5], device="cuda"))
    torch.cuda.synchronize()
