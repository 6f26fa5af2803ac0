"""What a row of attention makes of scales of values that are far from one another: those that it does not see have no part in it, and those that it
sees count by what they add, against 64 bits."""
import math

import numpy as np
import pytest
import torch

from tests.test_gpu_kv_attention import check as check_at, make, sampler  # noqa: F401
from tests import kv_oracle as oracle

pytestmark = pytest.mark.gpu


def rows(cache, q, table, start, kv_len, window=0):
    """{token: (out [Hq, D], bound)} in 64 bits. As kv_oracle.attention's bound, but what weights lose that are far below the largest is
    relative to the row's own largest weight: in units of which that one is 2^7 at least, fp16 below 2^-14 is off by 2^-25, so by 2^-32 of the
    largest weight for each key, times a code of up to 448. The largest weight's key has a code of 448 / 4 or more here: 2^-30 of
    that key's largest number. A unit is 2^-126 of the largest probability at least: 2^-25 of it each, 2^-151, times 448."""
    heads, page, dim = cache.k.shape[1], cache.k.shape[2], q.shape[2]
    group = q.shape[1] // heads
    wide = lambda x, s: x.float().cpu().double() * s.double().cpu().view(*s.shape, 1, 1)  # noqa: E731
    k_all, v_all, x_all = wide(cache.k, cache.k_scale), wide(cache.v, cache.v_scale), q.double().cpu()
    for i in range(len(kv_len)):
        first, last, n = int(start[i]), int(start[i + 1]), int(kv_len[i])
        pages = table[i, :-(-n // page)].astype(np.int64)
        k = k_all[pages].transpose(0, 1).reshape(heads, -1, dim)[:, :n]
        v = v_all[pages].transpose(0, 1).reshape(heads, -1, dim)[:, :n]
        for t in range(first, last):
            pos = n - (last - first) + t - first
            see = slice(max(0, pos + 1 - window) if window else 0, pos + 1)
            kk, vv = k[:, see], v[:, see]
            x = x_all[t].view(heads, group, dim)
            score = torch.einsum("hgd,hnd->hgn", x, kk) / math.sqrt(dim)
            size = (torch.einsum("hgd,hnd->hgn", x.abs(), kk.abs()) / math.sqrt(dim)).amax(2, keepdim=True)
            p = torch.softmax(score, 2)
            o, mass = p @ vv, p @ vv.abs()
            n_seen = kk.shape[1]
            weight = (p * vv.abs().amax(2).unsqueeze(1)).amax(2, keepdim=True)
            e = oracle.half_ulp(q.dtype) * o.abs() + torch.finfo(q.dtype).tiny * torch.finfo(q.dtype).eps
            e = e + (2.0 ** -11 + 2 * size * dim * 2.0 ** -23 + 2.0 ** -19 + (n_seen / 16 + 64) * 2.0 ** -22) * mass
            e = e + n_seen * (2.0 ** -30 * weight + 2.0 ** -151 * 448)
            yield t, o.reshape(-1, dim), (e * (1 + 2.0 ** -7)).reshape(-1, dim)


def check(sampler, cache, q, table, start, kv_len, window=0):  # noqa: F811
    cuda = lambda x: torch.from_numpy(x).cuda()  # noqa: E731
    out = sampler.kv_attention(q, cache, cuda(table), cuda(start), cuda(kv_len), max_new=int(np.diff(start).max()), window=window).double().cpu()
    for t, want, bound in rows(cache, q, table, start, kv_len, window):
        large = want.abs() + bound >= torch.finfo(q.dtype).max
        off = torch.where(large, 0.0, (out[t] - want).abs() / bound)
        assert (off <= 1).all(), (t, float(off.max()))
        assert (out[t].isfinite() | large).all(), t
    return out


@pytest.mark.parametrize("far", [20, 40, 90])
@pytest.mark.parametrize("page", [16, 24])
@pytest.mark.parametrize("kv_len,new,q_heads,dim", [([290, 300], 4, 4, 128), ([290, 130], 5, 8, 64), ([300, 310], 40, 8, 128), ([600, 310], 70, 4, 64)])
def test_scales_that_a_row_does_not_see(sampler, kv_len, new, q_heads, dim, page, far):  # noqa: F811
    """The last page's are 2^far times as large: rows in front of it do not see it, of the same block of keys or not. Then the first pages' of a
    window, which later rows do not see."""
    rng = np.random.default_rng(far + page)
    for window in (0, 60):
        cache, q, table, start, lens = make(rng, kv_len, [new] * 2, 2, q_heads, dim, page, "bf16")
        for i, n in enumerate(kv_len):
            # the last page that begins within the pass; in a window the page that its first row's window begins in
            at = (n - 1) // page if window == 0 else max(0, n - new + 1 - window + 2) // page
            cache.v_scale[int(table[i, at])] *= 2.0 ** far
        check(sampler, cache, q, table, start, lens, window)


@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("page", [16, 24])
@pytest.mark.parametrize("last", [False, True])
def test_scales_that_hardly_count(sampler, new, page, last):  # noqa: F811
    """A page whose keys have next to no weight and whose values are as much larger, before and behind the others; and one that has even less."""
    rng = np.random.default_rng(page)
    for up in (60, 40, 0):
        cache, q, table, start, lens = make(rng, [333], [new], 1, 4, 128, page, "bf16")
        q[:] = 1.5 + q * 0.02
        at = int(table[0, (333 - new) // page - 1 if last else 0])
        cache.k[at] = torch.full_like(cache.k[at].float(), -2.5).to(cache.k.dtype)  # a score of -42, 2^-61
        cache.k_scale[at] = 1.0
        cache.v_scale[at] *= 2.0 ** up
        check(sampler, cache, q, table, start, lens)


@pytest.mark.parametrize("new", [1, 3, 40])
@pytest.mark.parametrize("page", [16, 24])
@pytest.mark.parametrize("scale", [-100, -122, -126, -140, 100, 108])
def test_the_smallest_and_largest_scales(sampler, new, page, scale):  # noqa: F811
    rng = np.random.default_rng(new)
    cache, q, table, start, lens = make(rng, [150, 61], [new, new], 2, 8, 64, page, "bf16")
    cache.v_scale[:] = 2.0 ** scale
    out = check(sampler, cache, q, table, start, lens)
    assert scale == -140 or (out[:int(start[-1])] != 0).any(2).all()
    cache.v_scale[::2] = 2.0 ** (scale + 9 if scale < 0 else scale - 100)
    check(sampler, cache, q, table, start, lens)


@pytest.mark.parametrize("new", [1, 3, 40])
@pytest.mark.parametrize("page", [16, 24])
@pytest.mark.parametrize("up,of_scale", [(114, False), (117, False), (120, True), (124, False), (-85, False)])
def test_the_largest_and_smallest_queries(sampler, new, page, up, of_scale):  # noqa: F811
    """Rows up to the type's largest numbers, with keys or a scale of scores that make scores of their products."""
    rng = np.random.default_rng(up + 200)
    cache, q, table, start, lens = make(rng, [150, 61], [new, new], 2, 8, 128, page, "bf16")
    q.clamp_(-7.0, 7.0)  # 7 * 2^124 is a number
    q[1:, ::3] *= 2.0 ** -20
    q *= 2.0 ** up
    if not of_scale:
        cache.k_scale *= 2.0 ** (-up if up < 116 else -116)
    check_at(sampler, cache, q, table, start, lens, scale=2.0 ** (-up) / math.sqrt(128) if of_scale else 2.0 ** min(0, 116 - up) / math.sqrt(128))
