"""Attention over the paged 8-bit cache against 64 bits."""
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


def make(rng, kv_len, new, heads, q_heads, dim, page, kind, spare=3, q_size=1.5):
    """A cache, queries with rows of padding behind them, and the plan's arrays."""
    from mako_b200 import KvCache
    kv_len, new = np.asarray(kv_len), np.asarray(new)
    held = -(-kv_len // page)
    pages, cols = int(held.sum()) + spare, max(1, int(held.max(initial=0)))
    ids = rng.permutation(pages).astype(np.int32)
    table = np.full((len(kv_len), cols), -1, np.int32)
    at = 0
    for i, n in enumerate(held):
        table[i, :n] = ids[at:at + n]
        at += n
    cache = KvCache.empty(pages, heads, page, dim)
    for x, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        x.copy_(torch.from_numpy(rng.normal(0, 100, x.shape).astype(np.float32)).clamp(-448, 448).to(oracle.E4M3))
        s.copy_(torch.from_numpy(2.0 ** rng.integers(-9, -5, s.shape)).float())
        # places behind the last token hold anything
        for i, n in enumerate(kv_len):
            if n % page:
                x.view(torch.uint8)[int(table[i, held[i] - 1]), :, int(n % page):] = 0x7f
        x.view(torch.uint8)[torch.from_numpy(ids[at:].astype(np.int64)).cuda()] = 0xff
    start = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    q = torch.from_numpy(rng.normal(0, q_size, (int(start[-1]) + 2, q_heads, dim)).astype(np.float32)).to(TYPES[kind]).cuda()
    return cache, q, table, start, kv_len.astype(np.int32)


def check(sampler, cache, q, table, start, kv_len, window=0, scale=None, max_new=None, out=None, tokens=None):
    out = torch.full_like(q, 7.0) if out is None else out
    cuda = lambda x: torch.from_numpy(np.asarray(x, np.int32)).cuda()  # noqa: E731
    most = int(np.diff(start).max(initial=0)) if max_new is None else max_new
    sampler.kv_attention(q, cache, cuda(table), cuda(start), cuda(kv_len), max_new=most, scale=scale, window=window, out=out)
    wide = lambda x, s: x.float().cpu().double() * s.double().cpu().view(*s.shape, 1, 1)  # noqa: E731
    scale = 1 / math.sqrt(q.shape[2]) if scale is None else scale
    want, bound = oracle.attention(q.double().cpu(), wide(cache.k, cache.k_scale), wide(cache.v, cache.v_scale), table, start, kv_len,
                                   cache.k.shape[2], scale, window, q.dtype)
    got = out.double().cpu()
    rows = range(q.shape[0]) if tokens is None else tokens
    for t in rows:
        if t in want:
            a, b = got[t], want[t]
            assert torch.equal(a.isnan(), b.isnan()), t
            # a result beyond the type's largest number rounds to infinity of its sign
            large = (b.abs() + bound[t] >= torch.finfo(q.dtype).max) & a.isinf() & (a.sign() == b.sign())
            off = torch.where(large, 0.0, (a - b).abs().nan_to_num(0.0) - bound[t].nan_to_num(0.0))
            assert (off <= 0).all(), (t, float(off.max()), float(bound[t].max()))
        else:
            assert (got[t] == 7.0).all(), t
    return out


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("heads,q_heads,dim,page", [(1, 1, 128, 16), (2, 8, 128, 16), (2, 14, 64, 24), (1, 16, 128, 1), (3, 3, 64, 128), (1, 5, 128, 7),
                                                    (1, 24, 128, 32), (2, 64, 64, 16), (1, 50, 128, 16), (1, 130, 64, 40)])
@pytest.mark.parametrize("window", [0, 50])
def test_single_tokens(sampler, kind, heads, q_heads, dim, page, window):
    rng = np.random.default_rng(heads * 100 + q_heads + page)
    kv_len = [1, 2, 15, 16, 17, 0, 31, 33, 64, 100, 257, 500, 7]
    new = [1] * 13
    new[5] = 0
    check(sampler, *make(rng, kv_len, new, heads, q_heads, dim, page, kind), window=window)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("heads,q_heads,dim,page", [(1, 1, 128, 16), (2, 8, 128, 32), (1, 7, 64, 24), (2, 6, 128, 100)])
@pytest.mark.parametrize("window", [0, 20])
def test_rounds_and_chunks(sampler, kind, heads, q_heads, dim, page, window):
    rng = np.random.default_rng(heads * 100 + q_heads + page)
    kv_len, new = [5, 8, 40, 129, 64, 300, 1, 260], [5, 3, 2, 1, 4, 5, 1, 5]
    check(sampler, *make(rng, kv_len, new, heads, q_heads, dim, page, kind), window=window)
    kv_len, new = [150, 8, 40, 400, 0, 300, 1, 700], [150, 3, 33, 129, 0, 1, 1, 260]
    check(sampler, *make(rng, kv_len, new, heads, q_heads, dim, page, kind), window=window)


@pytest.mark.parametrize("q_heads", [2, 8, 40])
@pytest.mark.parametrize("dim", [64, 128])
def test_long_axis_is_split(sampler, q_heads, dim):
    """One sequence over many CTAs, and others whose units a cut goes through."""
    rng = np.random.default_rng(q_heads)
    check(sampler, *make(rng, [9001], [1], 2, q_heads, dim, 16, "bf16"))
    check(sampler, *make(rng, [3000, 40, 5001, 7, 1200], [1, 1, 2, 1, 3], 2, q_heads, dim, 16, "fp16"))


@pytest.mark.parametrize("dim,page,window", [(128, 16, 0), (64, 64, 1000), (128, 40, 0), (64, 7, 333)])
def test_long_prompts(sampler, dim, page, window):
    """Chunks over long contexts, whose units many CTAs share, beside single tokens and short ones; pages that are a multiple of 16 and not."""
    rng = np.random.default_rng(dim + page)
    check(sampler, *make(rng, [3000, 40, 1700, 129, 900], [300, 1, 130, 129, 17], 2, 10, dim, page, "bf16"), window=window)
    check(sampler, *make(rng, [2600], [65], 1, 4, dim, page, "fp16"), window=window)


@pytest.mark.parametrize("scale", [0.0, -0.05, 1e-30])
@pytest.mark.parametrize("new", [1, 40])
def test_scales_of_scores(sampler, scale, new):
    rng = np.random.default_rng(21)
    check(sampler, *make(rng, [300, 77], [new, new], 2, 8, 128, 16, "bf16"), scale=scale)


@pytest.mark.parametrize("rows", [16, 17, 63, 64, 65, 128, 129, 256, 257])
def test_rows_around_the_tiles(sampler, rows):
    """A key head's rows, at the borders of tiles, units and kernels, as tokens and as heads."""
    rng = np.random.default_rng(rows)
    check(sampler, *make(rng, [rows + 40, 3, rows], [rows, 1, rows], 1, 1, 64, 16, "bf16"))
    check(sampler, *make(rng, [150, 1, 33], [1, 1, 1], 1, rows, 64, 16, "fp16"))


def test_many_sequences(sampler):
    rng = np.random.default_rng(8)
    n = 700
    kv_len = rng.integers(0, 90, n)
    new = np.minimum(rng.integers(0, 3, n), kv_len)
    check(sampler, *make(rng, kv_len, new, 2, 4, 64, 16, "bf16"))


def test_a_row_that_sees_nothing_is_zeros(sampler):
    """No keys; more tokens than keys; pages that the table does not have, or that are none."""
    rng = np.random.default_rng(9)
    cache, q, table, start, kv_len = make(rng, [20, 40, 0, 3], [2, 1, 1, 5], 1, 4, 128, 16, "bf16")
    out = check(sampler, cache, q, table, start, kv_len)
    assert (out[3] == 0).all() and (out[4:6] == 0).all()
    table[0, 0], table[1, 1] = -1, 10 ** 6
    check(sampler, cache, q, table, start, kv_len)
    table[:] = -7
    assert (check(sampler, cache, q, table, start, kv_len)[:9] == 0).all()
    kv_len[:] = [1000, -5, 7, 2 ** 31 - 1]  # more than the table's pages
    check(sampler, cache, q, table, start, kv_len)


def test_rows_behind_the_last_sequence_and_wrong_starts(sampler):
    """Nothing beyond the rows of q is read or written, whatever the starts are."""
    rng = np.random.default_rng(10)
    cache, q, table, start, kv_len = make(rng, [20, 40, 33], [2, 1, 3], 1, 4, 64, 16, "fp16")
    for bad in ([0, 2, 3, 1000], [0, -7, 3, 4], [5, 3, 1, 0], [900, 901, 902, 2 ** 31 - 1]):
        cuda = lambda x: torch.from_numpy(np.asarray(x, np.int32)).cuda()  # noqa: E731
        sampler.kv_attention(q, cache, cuda(table), cuda(bad), cuda(kv_len), max_new=3)
    torch.cuda.synchronize()
    check(sampler, cache, q, table, start, kv_len)


@pytest.mark.parametrize("max_new", [0, 1, 5, 10 ** 6])
def test_max_new_chooses_nothing_but_kernels(sampler, max_new):
    rng = np.random.default_rng(11)
    check(sampler, *make(rng, [60, 41, 500], [9, 1, 70], 2, 8, 128, 16, "bf16"), max_new=max_new)


@pytest.mark.parametrize("new", [1, 4, 40])
def test_numbers_that_are_none(sampler, new):
    """A key or a value that is NaN is one for the rows that see it, and for no others; so is a query."""
    rng = np.random.default_rng(12)
    cache, q, table, start, kv_len = make(rng, [70, 70, 70], [new] * 3, 1, 4, 128, 16, "bf16")
    raw_v, raw_k = cache.v.view(torch.uint8), cache.k.view(torch.uint8)
    raw_k[int(table[0, 4]), 0, 5] = 0x7f   # key 69, which the last token alone sees
    raw_v[int(table[1, 4]), 0, 5] = 0xff   # value 69
    q[int(start[2]), 1, 7] = float("nan")
    check_nan = sampler.kv_attention(q, cache, *(torch.from_numpy(x).cuda() for x in (table, start, kv_len)), max_new=new)
    nan = check_nan.isnan().any(2).cpu()
    for i in range(3):
        rows = nan[int(start[i]):int(start[i + 1])]
        if i < 2:
            assert rows[-1].all() and not rows[:-1].any(), i
        else:
            assert rows[0].tolist() == [False, True, False, False] and not rows[1:].any()
    # in the middle of a window
    cache, q, table, start, kv_len = make(rng, [200], [new], 1, 4, 128, 16, "bf16")
    cache.v.view(torch.uint8)[int(table[0, 3]), 0, 3] = 0x7f  # value 51
    r = sampler.kv_attention(q, cache, *(torch.from_numpy(x).cuda() for x in (table, start, kv_len)), max_new=new, window=200 - new - 50)
    nan = r.isnan().any(2).cpu().numpy()[:new]
    sees = np.array([51 > 200 - new + t - (200 - new - 50) for t in range(new)])
    assert np.array_equal(nan.all(1), sees) and np.array_equal(nan.any(1), sees)


@pytest.mark.parametrize("kind", TYPES)
def test_large_and_small_numbers(sampler, kind):
    """Scores of thousands, rows of queries that differ by powers of two, scales of values that differ by 2^20."""
    rng = np.random.default_rng(13)
    cache, q, table, start, kv_len = make(rng, [300, 50, 129], [1, 1, 3], 2, 8, 128, 16, kind)
    q *= 30
    check(sampler, cache, q, table, start, kv_len)
    cache, q, table, start, kv_len = make(rng, [300, 50, 129], [1, 1, 3], 2, 8, 128, 16, kind)
    q[:, ::2] *= 2.0 ** -10
    if kind == "bf16":
        q[:, 1] *= 2.0 ** 60
        cache.k_scale *= 2.0 ** -60
        q[:, 3] *= 2.0 ** -60
    cache.v_scale[::3] *= 2.0 ** 20
    cache.v_scale[1::3] = 0.0
    check(sampler, cache, q, table, start, kv_len)


def test_scales_of_any_size(sampler):
    """A scale need not be a power of two."""
    rng = np.random.default_rng(14)
    cache, q, table, start, kv_len = make(rng, [300, 50], [1, 2], 2, 8, 64, 24, "fp16")
    cache.k_scale.uniform_(0.001, 0.01)
    cache.v_scale.uniform_(0.001, 0.01)
    check(sampler, cache, q, table, start, kv_len, scale=0.2)


def test_strides(sampler):
    """Queries that are a slice of a projection, an output with space between its rows, heads of the cache side by side."""
    from mako_b200 import KvCache
    rng = np.random.default_rng(15)
    cache, q, table, start, kv_len = make(rng, [300, 50, 77], [1, 2, 30], 2, 8, 128, 24, "bf16")
    wide = torch.randn(q.shape[0], 12, 128, device="cuda").bfloat16()
    wide[:, 2:10] = q
    out = torch.full((q.shape[0], 10, 128), 7.0, device="cuda").bfloat16()
    both = torch.zeros(cache.k.shape[0], 24, 2, 2, 128, dtype=torch.uint8, device="cuda").view(oracle.E4M3)
    other = KvCache(both[:, :, 0].transpose(1, 2), both[:, :, 1].transpose(1, 2), cache.k_scale, cache.v_scale)
    other.k.view(torch.uint8).copy_(cache.k.view(torch.uint8))
    other.v.view(torch.uint8).copy_(cache.v.view(torch.uint8))
    check(sampler, other, wide[:, 2:10], table, start, kv_len, out=out[:, 1:9])
    assert (out[:, 0] == 7).all() and (out[:, 9] == 7).all()
    one = check(sampler, cache, q[:1], table[:1], start[:2], kv_len[:1])
    assert one.shape == (1, 8, 128)


def test_streams_graphs_and_two_calls_at_once(sampler):
    rng = np.random.default_rng(16)
    sides = [make(rng, [5000, 700, 33], [1, 1, 1], 2, 8, 128, 16, "bf16"), make(rng, [4000, 90, 3000], [2, 50, 1], 2, 8, 128, 16, "bf16")]
    cuda = [[c, q] + [torch.from_numpy(x).cuda() for x in rest] for c, q, *rest in sides]
    call = lambda c, q, table, start, length, m: sampler.kv_attention(q, c, table, start, length, max_new=m, out=torch.zeros_like(q))  # noqa: E731
    want = [call(*x, m) for x, m in zip(cuda, (1, 50))]
    torch.cuda.synchronize()
    streams, graphs, got = [torch.cuda.Stream() for _ in sides], [], []
    for x, m, stream in zip(cuda, (1, 50), streams):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            got.append(call(*x, m))
        graphs.append(g)
    for _ in range(5):
        for g, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                g.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)
            a.zero_()
        torch.cuda.synchronize()


@pytest.mark.parametrize("new", [3, 40])
def test_pages_far_into_a_cache(sampler, new):
    """Offsets beyond 32 bits: 5.1 GB of keys and as many of values."""
    from mako_b200 import KvCache
    rng = np.random.default_rng(17)
    small, q, table, start, kv_len = make(rng, [100, 41], [1, new], 1, 4, 128, 16, "bf16")
    want = check(sampler, small, q, table, start, kv_len)
    pages = 2_500_000
    codes = lambda: torch.empty(pages, 1, 16, 128, dtype=torch.uint8, device="cuda").view(oracle.E4M3)  # noqa: E731
    big = KvCache(codes(), codes(), torch.ones(pages, 1, device="cuda"), torch.ones(pages, 1, device="cuda"))
    far = np.where(table >= 0, table.astype(np.int64) * 200_000 + 50_000, -1).astype(np.int32)
    for x, y in ((big.k, small.k), (big.v, small.v)):
        for i in range(small.k.shape[0]):
            x.view(torch.uint8)[i * 200_000 + 50_000] = y.view(torch.uint8)[i]
    for x, y in ((big.k_scale, small.k_scale), (big.v_scale, small.v_scale)):
        for i in range(small.k.shape[0]):
            x[i * 200_000 + 50_000] = y[i]
    got = sampler.kv_attention(q, big, *(torch.from_numpy(x).cuda() for x in (far, start, kv_len)), max_new=new, out=torch.full_like(q, 7.0))
    assert torch.equal(got, want)
