"""Rotated keys and values in the paged cache against 64 bits."""
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


def runs_of(rng, pages, page, lengths):
    """Slots of sequences that go on where they were (a place in a page) over pages of their own, rows of padding between and behind."""
    free = list(rng.permutation(pages))
    slots = []
    for place, n in lengths:
        p = free.pop()
        for _ in range(n):
            slots.append(int(p) * page + place)
            place += 1
            if place == page:
                place, p = 0, free.pop()
        slots += [-1] * int(rng.integers(0, 2))
    return np.array(slots + [-1, pages * page, -1], np.int64)


def cache_of(rng, pages, heads, page, dim, device="cuda"):
    from mako_b200 import KvCache
    c = KvCache.empty(pages, heads, page, dim, device)
    for x, s in ((c.k, c.k_scale), (c.v, c.v_scale)):
        x.copy_(torch.from_numpy(rng.normal(0, 100, x.shape)).clamp(-448, 448).float().to(oracle.E4M3))
        s.copy_(torch.from_numpy(2.0 ** rng.integers(-12, -6, s.shape)).float())
    return c


def check(sampler, cache, qkv, heads, q_heads, slots, positions, rotary, interleaved=False, scale=1.0, in_place=False):
    """qkv [T, q_heads + 2 heads, D] on the GPU."""
    t, page = len(slots), cache.k.shape[2]
    freq = torch.from_numpy((10000.0 ** (-np.arange(rotary // 2) * 2.0 / max(rotary, 1))).astype(np.float32))
    x = qkv.double().cpu().numpy()
    k0, v0 = cache.k.double().cpu().numpy(), cache.v.double().cpu().numpy()
    ks, vs = cache.k_scale.double().cpu().numpy(), cache.v_scale.double().cpu().numpy()
    q = qkv[:, :q_heads] if q_heads else None
    into = q if in_place else torch.full((t, q_heads, x.shape[2]), 7.0, dtype=qkv.dtype, device="cuda") if q_heads else None
    kw = dict(positions=torch.from_numpy(positions.astype(np.int32)).cuda(), inv_freq=freq.cuda(), interleaved=interleaved, rotary_scale=scale) if rotary else {}
    out = sampler.kv_append(cache, qkv[:, q_heads:q_heads + heads], qkv[:, q_heads + heads:], torch.from_numpy(slots).cuda(), q=q, q_out=into, **kw)
    turned, weight = x.copy(), np.zeros_like(x)
    for i in range(t):
        if rotary:
            turned[i, :q_heads + heads], weight[i, :q_heads + heads] = oracle.rotate(x[i, :q_heads + heads], float(positions[i]), freq.double().numpy(), interleaved, scale)
    real = (slots >= 0) & (slots < cache.k.shape[0] * page)
    # a rotated number: four roundings of 2^-24, a cosine and a sine of 2^-23 each
    room = 2.0 ** -21 * weight
    if q_heads:
        got = out.double().cpu().numpy()
        e = oracle.half_ulp(qkv.dtype) * np.abs(turned[:, :q_heads]) + room[:, :q_heads] * 1.01 + torch.finfo(qkv.dtype).tiny * torch.finfo(qkv.dtype).eps
        with np.errstate(invalid="ignore"):
            good = (np.abs(got - turned[:, :q_heads]) <= e) | (np.isnan(got) & ~np.isfinite(turned[:, :q_heads])) | (got == turned[:, :q_heads])
        assert good[real].all()
        left = x[:, :q_heads] if in_place else np.full_like(got, 7.0)
        assert np.array_equal(got[~real], left[~real], equal_nan=True)
    keys, values = turned[:, q_heads:q_heads + heads], turned[:, q_heads + heads:]
    fresh = np.zeros(k0.shape, bool)
    for s in slots[real]:
        fresh[s // page, :, s % page] = True
    # values are not rotated: every code and scale exactly
    wv, wvs = v0.copy(), vs.copy()
    oracle.append(wv, wvs, values, slots, page)
    assert np.array_equal(cache.v_scale.double().cpu().numpy(), wvs)
    assert np.array_equal(cache.v.double().cpu().numpy(), wv, equal_nan=True)
    # keys: scales but where the largest is next to a border, old codes exactly, new ones to half a step
    wk, wks = k0.copy(), ks.copy()
    oracle.append(wk, wks, keys, slots, page)
    low, high = ks.copy(), ks.copy()
    oracle.append(k0.copy(), low, keys * (1 - 2.0 ** -19), slots, page)
    oracle.append(k0.copy(), high, keys * (1 + 2.0 ** -19), slots, page)
    got_s, got = cache.k_scale.double().cpu().numpy(), cache.k.double().cpu().numpy()
    sure = low == high
    assert sure.mean() > 0.9 and np.array_equal(got_s[sure], wks[sure])
    old = ~fresh & np.broadcast_to(sure[:, :, None, None], k0.shape)
    assert np.array_equal(got[old], wk[old], equal_nan=True)
    for i in np.flatnonzero(real):
        p, at = slots[i] // page, slots[i] % page
        for h in np.flatnonzero(sure[p]):
            s = wks[p, h]
            step = np.maximum(np.abs(keys[i, h]) * 2.0 ** -4, s * 2.0 ** -10)
            y = got[p, h, at] * s
            with np.errstate(invalid="ignore"):
                good = (np.abs(y - keys[i, h]) <= step * (1 + 2.0 ** -10) + room[i, q_heads + h]) | (np.isnan(y) & ~np.isfinite(keys[i, h]))
            assert good.all(), (i, h)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("heads,q_heads,dim,rotary,page", [(1, 1, 64, 64, 16), (2, 8, 128, 128, 16), (3, 3, 64, 16, 7), (5, 10, 128, 64, 1),
                                                           (2, 0, 16, 16, 5), (1, 2, 256, 256, 24), (4, 28, 64, 0, 128), (8, 8, 128, 32, 64),
                                                           (3, 6, 48, 32, 16), (1, 3, 80, 80, 20), (5, 5, 240, 16, 9)])
def test_runs(sampler, kind, interleaved, heads, q_heads, dim, rotary, page):
    rng = np.random.default_rng(heads * 1000 + dim + page)
    slots = runs_of(rng, 400 if page == 1 else 60, page, [(0, 1), (page - 1, 1), (page // 2, 3), (0, 2 * page), (page // 3, 40), (0, page), (page - 1, page + 2)])
    positions = rng.integers(0, 5000, len(slots))
    positions[:4] = [0, 1, 131072, 2000000]
    qkv = torch.from_numpy(rng.normal(0, 1, (len(slots), q_heads + 2 * heads, dim)).astype(np.float32)).to(TYPES[kind]).cuda()
    cache = cache_of(rng, 400 if page == 1 else 60, heads, page, dim)
    check(sampler, cache, qkv, heads, q_heads, slots, positions, rotary, interleaved, 1.2)


@pytest.mark.parametrize("page", [16, 300])
def test_scales_that_grow_and_do_not(sampler, page):
    """Tokens one at a time, each some times as large as the one before, then smaller ones, zeros, and the smallest numbers there are."""
    rng = np.random.default_rng(page)
    cache = cache_of(rng, 2, 2, page, 64)
    sizes = [1e-3, 1.0, 3.0, 0.5, 100.0, 0.0, 1e4, 1e-30, 448.0, 3.5, 2.0 ** 15, 65000.0, 1e-38, 1.0, 2.0, 0.0]
    for i, m in enumerate(sizes):
        x = torch.from_numpy(rng.normal(0, m, (1, 4, 64)).astype(np.float32)).to(torch.bfloat16).cuda()
        check(sampler, cache, x, 2, 0, np.array([page + i]), np.array([i]), 64)


def test_pages_taken_over(sampler):
    """A run at place 0 does not care what the page's scale was, NaN and zero among it."""
    rng = np.random.default_rng(1)
    cache = cache_of(rng, 4, 1, 8, 64)
    cache.k_scale[:, 0] = torch.tensor([float("nan"), 0.0, 1e30, 1.0])
    cache.v_scale[:, 0] = torch.tensor([float("nan"), 0.0, 1e30, 1.0])
    x = torch.from_numpy(rng.normal(0, 1, (32, 2, 64)).astype(np.float32)).half().cuda()
    slots = torch.arange(32).cuda()
    sampler.kv_append(cache, x[:, :1], x[:, 1:], slots)
    for s, part in ((cache.k_scale, x[:, :1]), (cache.v_scale, x[:, 1:])):
        want = [oracle.scale_for(float(part[8 * i:8 * i + 8].abs().max())) for i in range(4)]
        assert s[:, 0].tolist() == want


def test_zeros_and_numbers_that_are_none(sampler):
    rng = np.random.default_rng(2)
    cache = cache_of(rng, 8, 2, 4, 64)
    x = torch.zeros(16, 4, 64)
    x[4:8] = torch.randn(4, 4, 64)
    x[5, :, 3], x[6, :, 4], x[7, :, 5] = float("nan"), float("inf"), -float("inf")
    x[8:12] = float("nan")
    x[12:] = torch.randn(4, 4, 64) * 1e-20
    check(sampler, cache, x.bfloat16().cuda(), 2, 0, np.arange(16, dtype=np.int64), np.arange(16), 0)


def test_in_place_padding_and_nothing(sampler):
    rng = np.random.default_rng(3)
    cache = cache_of(rng, 10, 2, 16, 64)
    x = torch.from_numpy(rng.normal(0, 1, (20, 8, 64)).astype(np.float32)).half().cuda()
    slots = np.concatenate([[-1, -1], np.arange(30, 40), [-1], np.arange(64, 70), [10 ** 12]]).astype(np.int64)
    check(sampler, cache, x, 2, 4, slots, rng.integers(0, 99, 20), 64, in_place=True)
    check(sampler, cache, x, 2, 4, np.full(20, -1, np.int64), np.zeros(20), 64)
    before = cache.k.view(torch.uint8).clone()
    sampler.kv_append(cache, x[:0, :2], x[:0, 2:4], torch.zeros(0, dtype=torch.int64, device="cuda"))
    assert torch.equal(before, cache.k.view(torch.uint8))


@pytest.mark.parametrize("tokens", [1025, 5000])
def test_long_passes(sampler, tokens):
    rng = np.random.default_rng(4)
    page, dim = 32, 128
    cache = cache_of(rng, tokens // page + 3, 2, page, dim)
    x = torch.from_numpy(rng.normal(0, 1, (tokens, 6, dim)).astype(np.float32)).to(torch.bfloat16).cuda()
    check(sampler, cache, x, 2, 2, np.arange(tokens, dtype=np.int64) + 11, np.arange(tokens), 128)


@pytest.mark.parametrize("rotary", [0, 16])
def test_a_page_as_long_as_a_sequence(sampler, rotary):
    rng = np.random.default_rng(6)
    page, tokens = 70000, 66000
    cache = cache_of(rng, 2, 1, page, 16)
    x = torch.from_numpy(rng.normal(0, 1, (tokens, 4, 16)).astype(np.float32)).to(torch.float16).cuda()
    x[-1] *= 9.0  # the scales are the last row's
    check(sampler, cache, x, 1, 2, np.arange(tokens, dtype=np.int64) + page + 3000, np.arange(tokens), rotary)


def test_a_cache_whose_heads_stand_side_by_side(sampler):
    """[P, page, H, D] seen as its transpose, and both kinds in one allocation."""
    from mako_b200 import KvCache
    rng = np.random.default_rng(5)
    a = cache_of(rng, 6, 3, 8, 64)
    both = torch.zeros(6, 8, 2, 3, 64, dtype=torch.uint8, device="cuda").view(oracle.E4M3)
    b = KvCache(both[:, :, 0].transpose(1, 2), both[:, :, 1].transpose(1, 2), a.k_scale.clone(), a.v_scale.clone())
    b.k.view(torch.uint8).copy_(a.k.view(torch.uint8))
    b.v.view(torch.uint8).copy_(a.v.view(torch.uint8))
    x = torch.from_numpy(rng.normal(0, 2, (20, 6, 64)).astype(np.float32)).to(torch.bfloat16).cuda()
    slots = torch.arange(5, 25).cuda()
    for c in (a, b):
        sampler.kv_append(c, x[:, :3], x[:, 3:], slots)
    for k in ("k", "v"):
        assert torch.equal(getattr(a, k).view(torch.uint8), getattr(b, k).contiguous().view(torch.uint8))
    assert torch.equal(a.k_scale, b.k_scale) and torch.equal(a.v_scale, b.v_scale)
