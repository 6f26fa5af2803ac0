"""Log-probabilities of given tokens, entropies and alternatives against 64 bits."""
import numpy as np
import pytest
import torch

from tests import kv_oracle as oracle

pytestmark = pytest.mark.gpu
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


@pytest.fixture(scope="module")
def sampler():
    from mako_b200 import BatchSampler
    return BatchSampler(32, 1)


def pack(bits):
    words = -(-bits.shape[1] // 32)
    b = np.zeros((len(bits), words * 32), np.uint64)
    b[:, :bits.shape[1]] = bits
    return torch.from_numpy((b.reshape(len(bits), words, 32) << np.arange(32, dtype=np.uint64)).sum(2).astype(np.uint32).view(np.int32)).cuda()


def check(sampler, x, tokens, temperature, top, allowed=None, mask=None):
    t = torch.as_tensor(temperature, dtype=torch.float32)
    r = sampler.token_logprobs(x, tokens, t.cuda() if t.dim() else float(t), top=top, mask=pack(allowed) if mask is None and allowed is not None else mask)
    rows = x.double().cpu().numpy()
    want = tokens.cpu().numpy().reshape(len(rows), -1)
    got = [y.double().cpu().numpy() for y in (r.logprob, r.entropy, r.top_ids, r.top_logprobs)]
    given = got[0].reshape(len(rows), -1)
    for i in range(len(rows)):
        lp, h, ids, tops, bound, bound_h = oracle.logprobs(rows[i], want[i], float(t[i] if t.dim() else t), top, None if allowed is None else allowed[i])
        assert got[2][i].tolist() == ids.tolist(), i
        room = np.array([bound[k] if 0 <= k < len(bound) else 0.0 for k in want[i]])
        for a, b, e in ((given[i], lp, room), (got[3][i], tops, bound[ids])):
            same = (a == b) | (np.abs(a - np.where(np.isinf(b), 0, b)) <= e) & np.isfinite(b)
            assert same.all(), (i, a, b, e)
        assert abs(got[1][i] - h) <= bound_h, (i, got[1][i], h, bound_h)
        dead = not ((~np.isnan(rows[i])) & (rows[i] > -np.inf) & (True if allowed is None else allowed[i])).any()
        none = allowed is not None and not allowed[i].any()
        assert int(r.flags[i]) == (0x4 if dead else 0) + (0x8 if dead and none else 0)
    return r


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rows,vocab,top", [(1, 1, 1), (3, 7, 0), (2, 33, 20), (5, 1000, 64), (1, 50257, 5), (300, 4099, 20), (2, 129280, 64), (150, 9000, 1)])
def test_rows(sampler, kind, rows, vocab, top):
    rng = np.random.default_rng(vocab + rows)
    x = torch.from_numpy(rng.normal(0, 3, (rows, vocab)).astype(np.float32)).to(TYPES[kind]).cuda()
    tokens = torch.from_numpy(rng.integers(-1, vocab, (rows, 2)).astype(np.int32)).cuda()
    check(sampler, x, tokens, 0.7, top)


@pytest.mark.parametrize("given", [0, 33, 300, 1000])
@pytest.mark.parametrize("rows", [2, 500])
def test_many_tokens_of_a_row(sampler, rows, given):
    rng = np.random.default_rng(given)
    x = torch.from_numpy(rng.normal(0, 3, (rows, 9001)).astype(np.float32)).to(torch.bfloat16).cuda()
    tokens = torch.from_numpy(rng.integers(-1, 9001, (rows, given)).astype(np.int32)).cuda()
    check(sampler, x, tokens, 1.3, 5, rng.random((rows, 9001)) < 0.6)


@pytest.mark.parametrize("kind", TYPES)
def test_masks_and_temperatures_of_the_rows(sampler, kind):
    rng = np.random.default_rng(3)
    n, v = 9, 5003
    x = torch.from_numpy(rng.normal(0, 3, (n, v)).astype(np.float32)).to(TYPES[kind]).cuda()
    allowed = rng.random((n, v)) < np.linspace(0, 0.9, n)[:, None] ** 3
    allowed[2] = False
    allowed[2, 7] = True
    tokens = torch.from_numpy(rng.integers(0, v, (n, 3)).astype(np.int32)).cuda()
    tokens[2, 0] = 7
    check(sampler, x, tokens, [1.0, 0.5, 1.0, 0.0, 1e-3, 30.0, -1.0, 1e31, 2.0], 20, allowed)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("start", range(9))
def test_rows_at_any_element_with_masks(sampler, kind, start):
    rng = np.random.default_rng(start)
    n, v = 4, 1237
    x = torch.from_numpy(rng.normal(0, 3, (n, v + 20)).astype(np.float32)).to(TYPES[kind]).cuda()
    x[:, :start] = 50.0  # not the rows' own
    x[:, start + v:] = 50.0
    allowed = rng.random((n, v)) < 0.3
    tokens = torch.from_numpy(rng.integers(0, v, n).astype(np.int32)).cuda()
    check(sampler, x[:, start:start + v], tokens, 1.0, 9, allowed)
    check(sampler, x[:, start:start + v], tokens, 1.0, 9)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("vocab", [3000, 40000])
@pytest.mark.parametrize("shape", ["rising", "falling", "equal", "two", "steps"])
def test_orders_and_ties(sampler, kind, vocab, shape):
    """Lists that run over, and equal logits: the lowest ids."""
    at = torch.arange(vocab, dtype=torch.float64)
    row = {"rising": at / vocab * 8, "falling": -at / vocab * 8, "equal": at * 0 + 1.5, "two": (at % 7 == 3).double(), "steps": (at / 600).floor() % 5}[shape]
    x = torch.stack([row, row.flip(0)]).to(TYPES[kind]).cuda()
    check(sampler, x, torch.tensor([[0], [vocab - 1]], dtype=torch.int32).cuda(), 1.0, 64)


@pytest.mark.parametrize("kind", TYPES)
def test_numbers_that_are_none_and_infinities(sampler, kind):
    inf, nan = float("inf"), float("nan")
    v, n = 2500, 9
    x = torch.randn(n, v, generator=torch.Generator().manual_seed(1)).double()
    x[0, 5], x[0, 2000:] = nan, nan
    x[1, 9], x[1, 400] = inf, inf
    x[2] = -inf
    x[3] = nan
    x[4, 3:] = -inf
    x[5] = -inf
    x[5, 11] = 2.0
    x[6, ::2] = torch.finfo(TYPES[kind]).min
    x[7] = torch.finfo(TYPES[kind]).min
    x[8, 100], x[8, 200] = inf, nan
    tokens = torch.tensor([[5, 3], [400, 9], [0, 1], [7, 8], [1, 900], [11, 12], [2, 3], [0, 5], [200, 100]], dtype=torch.int32).cuda()
    check(sampler, x.to(TYPES[kind]).cuda(), tokens, 1.0, 5)


def test_tokens_outside_of_the_vocabulary_name_none(sampler):
    x = torch.randn(2, 100, device="cuda")
    r = sampler.token_logprobs(x, torch.tensor([-5, 100], dtype=torch.int32).cuda())
    assert r.logprob.tolist() == [0.0, 0.0] and r.top_ids.shape == (2, 0)


def test_what_is_behind_the_results_stays(sampler):
    """Rows with and without alternatives, and no rows at all."""
    x = torch.randn(0, 100, device="cuda")
    r = sampler.token_logprobs(x, torch.zeros(0, dtype=torch.int32, device="cuda"), top=3)
    assert r.logprob.shape == (0,) and r.top_ids.shape == (0, 3)


def test_a_far_row(sampler):
    """Offsets beyond 32 bits: 2.2e9 elements into the rows."""
    n, v = 2200, 1_000_003
    x = torch.empty(n, v, dtype=torch.bfloat16, device="cuda")
    x[:2] = 0
    x[-2:] = torch.randn(2, v, device="cuda")
    last = x[-2:]
    base = sampler.token_logprobs(last.clone(), torch.tensor([5, 6], dtype=torch.int32).cuda(), top=4)
    rows = x.as_strided((2, v), ((n - 1) * v, 1))
    got = sampler.token_logprobs(rows, torch.tensor([5, 6], dtype=torch.int32).cuda(), top=4)
    assert torch.equal(got.logprob[1], base.logprob[1]) and torch.equal(got.top_ids[1], base.top_ids[1])


def test_streams_graphs_and_repeated_calls(sampler):
    x, tokens = torch.randn(40, 30000, device="cuda").half(), torch.randint(0, 30000, (40,), device="cuda", dtype=torch.int32)
    want = sampler.token_logprobs(x, tokens, 0.9, top=8)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=stream):
        got = sampler.token_logprobs(x, tokens, 0.9, top=8)
    for _ in range(3):
        got.logprob.zero_()
        g.replay()
        torch.cuda.synchronize()
        for k in ("logprob", "entropy", "top_ids", "top_logprobs", "flags"):
            assert torch.equal(getattr(got, k), getattr(want, k)), k


def test_beside_the_sampler(gpu_sampler_factory):
    """The log-probability of the token that an untruncated sample call draws is that of its probability."""
    from mako_b200 import SamplingParams
    s = gpu_sampler_factory(5000, 64)
    x = torch.randn(16, 5000, device="cuda") * 2
    drawn = s.sample(x, SamplingParams(temperature=0.8), torch.rand(16, device="cuda"))
    r = s.token_logprobs(x, drawn.token, 0.8, top=1)
    assert torch.allclose(r.logprob.exp(), drawn.prob, rtol=2e-5, atol=0)
