"""Attention of prompts over the paged cache where a CTA has many short units one behind the other, against 64 bits (on the GPU, a sequence at a
time): prompts from their first token, whose units are a block or two long."""
import math

import numpy as np
import pytest
import torch

from tests import kv_oracle as oracle

pytestmark = pytest.mark.gpu
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


@pytest.fixture(scope="module")
def sampler():
    from mako_b200 import BatchSampler
    return BatchSampler(32, 1)


def make(seed, kv_len, new, heads, group, dim, page, kind, spread=20, step=3):
    """A cache whose scales of values differ by up to 2^spread from one sequence and head to another, by up to 2^step among their pages."""
    from mako_b200 import KvCache
    g = torch.Generator(device="cuda").manual_seed(seed)
    rng = np.random.default_rng(seed)
    kv_len, new = np.asarray(kv_len), np.asarray(new)
    held = -(-kv_len // page)
    pages, cols = int(held.sum()), int(held.max())
    ids = rng.permutation(pages).astype(np.int32)
    table = np.full((len(kv_len), cols), -1, np.int32)
    of = np.zeros(pages, np.int64)  # a page's sequence
    at = 0
    for i, n in enumerate(held):
        table[i, :n] = ids[at:at + n]
        of[ids[at:at + n]] = i
        at += n
    cache = KvCache.empty(pages, heads, page, dim)
    for x in (cache.k, cache.v):
        x.copy_(torch.empty(x.shape, device="cuda").normal_(0, 100, generator=g).clamp_(-448, 448).to(oracle.E4M3))
    cache.k_scale.copy_(torch.from_numpy(2.0 ** rng.integers(-9, -5, (pages, heads))).float())
    base = rng.integers(-9 - spread, -8, (len(kv_len), heads))
    cache.v_scale.copy_(torch.from_numpy(2.0 ** (base[of] + rng.integers(0, step + 1, (pages, heads)))).float())
    start = np.concatenate([[0], np.cumsum(new)])
    q = torch.empty(int(start[-1]), heads * group, dim, device="cuda").normal_(0, 1.5, generator=g).to(TYPES[kind])
    return cache, q, table, start.astype(np.int32), kv_len.astype(np.int32)


def expected(cache, q, table, start, kv_len, window=0):
    """For each sequence: (first row, out, bound, sees_nan) with out and bound [n, heads, group, D], sees_nan [n, heads]. The bound is that
    of kv_oracle.attention."""
    page, dim = cache.k.shape[2], q.shape[2]
    heads, group = cache.k.shape[1], q.shape[1] // cache.k.shape[1]
    for i in range(len(kv_len)):
        first, last, n = int(start[i]), int(start[i + 1]), int(kv_len[i])
        if first == last:
            continue
        ids = torch.from_numpy(table[i, :-(-n // page)].astype(np.int64)).cuda()
        wide = lambda x, s: (x[ids].double() * s[ids].double().view(len(ids), heads, 1, 1)).transpose(0, 1).reshape(heads, -1, dim)[:, :n]  # noqa: E731
        k, v = wide(cache.k, cache.k_scale), wide(cache.v, cache.v_scale)
        bad = v.isnan().any(2)  # [heads, n]
        v = v.nan_to_num(0.0)
        x = q[first:last].double().view(-1, heads, group, dim)
        pos = n - (last - first) + torch.arange(last - first, device="cuda").view(-1, 1)
        key = torch.arange(n, device="cuda").view(1, -1)
        see = (key <= pos) & ((key > pos - window) if window else True)
        outs, bounds = [], []
        for h in range(heads):
            score = torch.einsum("tgd,nd->tgn", x[:, h], k[h]) / math.sqrt(dim)
            size = (torch.einsum("tgd,nd->tgn", x[:, h].abs(), k[h].abs()) / math.sqrt(dim)).masked_fill(~see[:, None], 0.0).amax(2, keepdim=True)
            p = torch.softmax(score.masked_fill(~see[:, None], -math.inf), 2)
            o, mass = p @ v[h], p @ v[h].abs()
            most = torch.where(see, v[h].abs().amax(1).view(1, -1), 0.0).amax(1).view(-1, 1, 1)
            count = see.sum(1).view(-1, 1, 1)
            tiny = 2.0 ** -30 * most * count * p.amax(2, keepdim=True)
            e = oracle.half_ulp(q.dtype) * o.abs() + torch.finfo(q.dtype).tiny * torch.finfo(q.dtype).eps
            e = e + (2.0 ** -11 + 2 * size * dim * 2.0 ** -23 + 2.0 ** -19 + (count / 16 + 64) * 2.0 ** -22) * mass + tiny
            outs.append(o)
            bounds.append(e * (1 + 2.0 ** -7))
        yield first, torch.stack(outs, 1), torch.stack(bounds, 1), (see[:, None] & bad).any(2)


def call(sampler, cache, q, table, start, kv_len, window=0):
    cuda = lambda x: torch.from_numpy(x).cuda()  # noqa: E731
    return sampler.kv_attention(q, cache, cuda(table), cuda(start), cuda(kv_len), max_new=int(np.diff(start).max()), window=window)


def check(sampler, cache, q, table, start, kv_len, window=0):
    out = call(sampler, cache, q, table, start, kv_len, window)
    heads = cache.k.shape[1]
    for first, want, bound, nan in expected(cache, q, table, start, kv_len, window):
        got = out[first:first + len(want)].double().view(want.shape)
        off = (got - want).abs() / bound
        assert (off.nan_to_num(0.0) <= 1).all(), (first, float(off.nan_to_num(0.0).max()))
        # a row that sees a value which is NaN is one (in its column at least), no other is
        assert torch.equal(got.isnan().any(3), nan.view(-1, heads, 1).expand(got.shape[:3])), first
    for _ in range(4):
        again = call(sampler, cache, q, table, start, kv_len, window)
        assert torch.equal(again.view(torch.int16), out.view(torch.int16))


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("low,high,group,dim,page,window", [(60, 128, 4, 128, 16, 0), (65, 128, 8, 64, 24, 0), (129, 256, 4, 64, 16, 0), (90, 128, 4, 128, 20, 40),
                                                            (65, 300, 5, 128, 32, 33)])
def test_many_short_prompts(sampler, kind, low, high, group, dim, page, window):
    rng = np.random.default_rng(low + high)
    n = rng.integers(low, high + 1, 70)
    check(sampler, *make(low + page, n, n, 8, group, dim, page, kind), window=window)


@pytest.mark.parametrize("page", [16, 24])
def test_values_that_are_none_in_short_prompts(sampler, page):
    """Every third sequence has a value that is NaN, which its last rows alone see."""
    rng = np.random.default_rng(page)
    n = rng.integers(65, 129, 80)
    cache, q, table, start, kv_len = make(page, n, n, 8, 4, 128, page, "bf16")
    raw = cache.v.view(torch.uint8)
    for i in range(0, 80, 3):
        at, h = int(n[i]) - 1 - int(rng.integers(0, 20)), int(rng.integers(0, 8))
        raw[int(table[i, at // page]), h, at % page, int(rng.integers(0, 128))] = 0x7f
    check(sampler, cache, q, table, start, kv_len)


def test_prompts_and_their_first_tokens(sampler):
    """Long prompts from their first token: the end of one head, then the first blocks of the next; short ones and chunks beside them."""
    check(sampler, *make(3, [2048] * 4 + [1000, 2048, 77, 2047], [2048] * 4 + [1000, 2048, 77, 2047], 8, 4, 128, 64, "bf16"))
    check(sampler, *make(4, [700, 90, 128, 1, 300, 128] * 12, [200, 90, 128, 1, 30, 100] * 12, 4, 8, 64, 16, "fp16"))
