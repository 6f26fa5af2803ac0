"""Speculative rounds against whole distributions (mk_spec_verify), against the 64-bit form."""
import math

import numpy as np
import pytest
import torch

from tests import round_oracle as oracle

pytestmark = pytest.mark.gpu

NEAR = 1e-9  # decisions closer than this may fall either way: u, P and Q are products of a few roundings of 2^-53 over rows of <= 2e5


def rows(rng, n, v, dtype, sigma=2.0):
    x = rng.normal(0.0, sigma, (n, v)).astype(np.float32)
    x[np.arange(n)[:, None], rng.integers(0, v, (n, 8))] = rng.uniform(8, 15, (n, 8))
    return torch.from_numpy(x).to(dtype)


def case(seed, s, d, v, dtype=torch.float32, onehot=False, mask=0.0, ragged=True, noise=0.7, sigma=2.0, mixed=True):
    rng = np.random.default_rng(seed)
    target = rows(rng, s * (d + 1), v, dtype, sigma)
    draft = (target.view(s, d + 1, v)[:, :d].float() + noise * torch.from_numpy(rng.normal(size=(s, d, v)).astype(np.float32)))
    draft = draft.reshape(s * d, v).to(dtype)
    t = rng.uniform(0.4, 1.3, s).astype(np.float32) if mixed else np.full(s, 0.8, np.float32)
    words = None
    if mask:
        b = rng.random((s * (d + 1), ((v + 31) // 32) * 32)) < mask
        words = np.packbits(b.reshape(len(b), -1, 32), axis=2, bitorder="little").view(np.uint32)[:, :, 0].astype(np.uint32)
    x = draft.float().numpy() / np.repeat(t, d)[:, None] if d else np.zeros((0, v), np.float32)
    if mask and d:
        x = np.where(b.reshape(s, d + 1, -1)[:, :d, :v].reshape(s * d, v), x, -np.inf)
    drafts = (x + rng.gumbel(size=x.shape)).argmax(1).reshape(s, d).astype(np.int32)
    if ragged and d:
        drafts[np.arange(d)[None] >= rng.integers(0, d + 1, (s, 1))] = -1
    return {"logits": target, "drafts": drafts, "u": rng.random((s, d + 2)).astype(np.float32), "temperature": t,
            "draft_logits": None if onehot else draft, "mask": words, "mask_drafts": bool(mask)}


def compare(sampler, c, pad=0, offset=0, **kw):
    """pad, offset: columns behind a row and in front of the first, so that rows start at any element."""
    def spread(x):
        if x is None:
            return None
        wide = torch.full((x.shape[0] * (x.shape[1] + pad) + offset,), math.nan, dtype=x.dtype, device="cuda")
        out = wide[offset:].view(x.shape[0], x.shape[1] + pad)[:, :x.shape[1]]
        out.copy_(x)
        return out
    want = oracle.verify(c["logits"].double().numpy(), c["drafts"], c["u"], c["temperature"],
                         None if c["draft_logits"] is None else c["draft_logits"].double().numpy(), c.get("draft_temperature"),
                         c["mask"], c["mask_drafts"])
    cuda = lambda x: None if x is None else torch.from_numpy(np.ascontiguousarray(x)).cuda()  # noqa: E731
    temperature = kw.get("temperature", cuda(c["temperature"]))
    got = sampler.spec_verify(spread(c["logits"]), cuda(c["drafts"]), cuda(c["u"]), temperature,
                              draft_logits=spread(c["draft_logits"]), draft_temperature=cuda(c.get("draft_temperature")),
                              mask=cuda(c["mask"].view(np.int32)) if c["mask"] is not None else None,
                              mask_drafts=c["mask_drafts"])
    kept, nxt, tokens, lp, flags = [x.cpu().numpy() for x in (got.n_kept, got.next_token, got.tokens, got.logprob, got.flags)]
    sure = 0
    for i, (j, t, toks, logs, f, margin) in enumerate(want):
        if margin < NEAR:
            continue
        sure += 1
        assert (kept[i], nxt[i], flags[i]) == (j, t, f), (i, kept[i], nxt[i], flags[i], j, t, f, margin)
        assert tokens[i].tolist() == toks, i
        # log P: a rounding to fp32, and what rows of fp32 exponentials leave of the sum
        assert np.allclose(lp[i], logs, rtol=2.0 ** -22, atol=2e-6), (i, lp[i], logs)
    # that few are passed over: a tenth, or one of a few (of far_from_one's eight rows one has a draft of 1.7e-299 of the whole, which
    # is less than the 1e-290 that weigh anything)
    assert sure >= len(want) - max(1, len(want) // 10)
    return got


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("s, d, v", [(1, 4, 129280), (1, 0, 50257), (5, 3, 32003), (40, 7, 4099), (300, 2, 1000), (3, 1, 33), (7, 2, 1)])
def test_sizes(gpu_sampler_factory, dtype, s, d, v):
    for onehot in (False, True):
        compare(gpu_sampler_factory(129280, 512), case(s * 100 + d, s, d, v, dtype, onehot))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("pad, offset", [(0, 1), (1, 0), (3, 2), (7, 5), (5, 0)])
def test_rows_start_anywhere(gpu_sampler_factory, dtype, pad, offset):
    """What lies between the rows is NaN and has no part in them."""
    c = case(77 + pad, 6, 3, 9001, dtype)
    compare(gpu_sampler_factory(129280, 512), c, pad, offset)
    compare(gpu_sampler_factory(129280, 512), case(78 + pad, 6, 3, 9001, dtype, True, mask=0.2), pad, offset)


@pytest.mark.parametrize("sigma", [0.0, 0.3, 6.0])
def test_flat_and_steep_rows(gpu_sampler_factory, sigma):
    c = case(int(sigma * 10), 12, 3, 100001, sigma=sigma, noise=0.1)
    if sigma == 0.0:  # wholly flat: every token as likely as the other
        c["logits"].zero_()
        c["draft_logits"].fill_(1.0)
    compare(gpu_sampler_factory(129280, 512), c)


@pytest.mark.parametrize("onehot", [False, True])
@pytest.mark.parametrize("fraction", [0.5, 0.02, 0.0005])
def test_masks(gpu_sampler_factory, fraction, onehot):
    """Masks down to a few tokens a row and to none, over the drafter's rows too or not."""
    c = case(int(fraction * 1e4), 24, 3, 20011, torch.float16, onehot, mask=fraction)
    if fraction < 0.001:
        c["mask"][5:9] = 0
        c["mask"][40] = 0
        c["mask"][41] = 0
        c["mask"][41, -1] = 0xfffffff8  # behind the last column
    compare(gpu_sampler_factory(129280, 512), c)
    c["mask_drafts"] = False
    compare(gpu_sampler_factory(129280, 512), c)


def test_greedy_and_draft_temperatures(gpu_sampler_factory):
    c = case(3, 30, 3, 5000)
    c["temperature"][::3] = 0.0
    c["temperature"][1::9] = -1.0
    c["temperature"][2] = 1e-3
    c["draft_temperature"] = np.random.default_rng(1).uniform(0.3, 2.0, 30).astype(np.float32)
    c["draft_temperature"][::4] = 0.0
    for i in range(30):
        if i % 2 == 0:
            c["drafts"][i, 0] = int(c["logits"][i * 4].argmax())
    compare(gpu_sampler_factory(129280, 512), c)
    c = case(4, 8, 2, 5000, mixed=False)
    compare(gpu_sampler_factory(129280, 512), c, temperature=float(c["temperature"][0]))
    c["temperature"][:] = 0.0
    compare(gpu_sampler_factory(129280, 512), c, temperature=0.0)


def test_infinities_nan_and_empty_rows(gpu_sampler_factory):
    """Logits of the type's lowest value, -inf, +inf and NaN anywhere; rows without a finite value; ties for the largest."""
    for dtype in (torch.float32, torch.bfloat16):
        c = case(9, 16, 2, 3001, dtype, ragged=False)
        x, q = c["logits"].view(16, 3, 3001), c["draft_logits"].view(16, 2, 3001)
        low = torch.finfo(dtype).min
        x[0, :, 5:] = low
        x[1, 0] = -math.inf
        x[2, 1] = math.nan
        x[3, :, ::3] = math.nan
        x[4, 0, 77] = math.inf
        x[4, 1, 78], x[4, 1, 99] = math.inf, math.inf
        q[5, 0] = -math.inf
        q[6, 0, 40] = math.inf
        q[7, :, ::2] = math.nan
        x[8, 0], q[8, 0] = -math.inf, math.nan
        x[9, 0] = low
        x[10, 0] = 0.0
        q[10, 0] = 0.0
        x[11] = q[11, :1]  # the same rows: always kept
        c["temperature"][9:11] = 0.0
        c["drafts"][12] = [3001, 5]
        c["drafts"][13] = [-5, 5]
        compare(gpu_sampler_factory(129280, 512), c)


def test_uniforms_at_the_ends(gpu_sampler_factory):
    for onehot in (False, True):
        c = case(15, 20, 3, 8000, onehot=onehot)
        c["u"][::2] = 0.0
        c["u"][1::2] = np.nextafter(np.float32(1), np.float32(0))
        cuda = lambda x: None if x is None else torch.as_tensor(x).cuda()  # noqa: E731
        got = gpu_sampler_factory(129280, 512).spec_verify(
            cuda(c["logits"]), cuda(c["drafts"]), cuda(c["u"]), cuda(c["temperature"]), draft_logits=cuda(c["draft_logits"]))
        n_drafts = (c["drafts"] >= 0).cumprod(1).sum(1)
        assert np.array_equal(got.n_kept.cpu().numpy()[::2], n_drafts[::2])  # 0 < P
        assert (got.next_token.cpu().numpy() >= 0).all() and (got.next_token.cpu().numpy() < 8000).all()


def test_the_drawn_tokens_follow_the_target(gpu_sampler_factory):
    """What a round yields first is distributed as the target, whatever the drafter: 60,000 rounds over eleven tokens."""
    rng = np.random.default_rng(2)
    n, v = 60000, 11
    t, q = rng.normal(0, 1.5, v).astype(np.float32), rng.normal(0, 1.5, v).astype(np.float32)
    p, qq = np.exp(t.astype(np.float64)), np.exp(q.astype(np.float64))
    p, qq = p / p.sum(), qq / qq.sum()
    from mako_b200 import BatchSampler
    sampler = BatchSampler(v, n)
    logits = torch.from_numpy(t).cuda().expand(2 * n, v).contiguous()
    draft = torch.from_numpy(q).cuda().expand(n, v).contiguous()
    drafts = torch.from_numpy(rng.choice(v, (n, 1), p=qq).astype(np.int32)).cuda()
    u = torch.from_numpy(rng.random((n, 3)).astype(np.float32)).cuda()
    got = sampler.spec_verify(logits, drafts, u, 1.0, draft_logits=draft)
    freq = np.bincount(got.tokens[:, 0].cpu().numpy(), minlength=v) / n
    assert np.all(np.abs(freq - p) < 5 * np.sqrt(p * (1 - p) / n))  # five standard deviations of a share of n draws


def test_streams_and_captures(gpu_sampler_factory):
    """On a stream of its own, and captured: two graphs of one handle, replayed one behind the other on new inputs."""
    sampler = gpu_sampler_factory(129280, 512)
    cuda = lambda x: None if x is None else torch.as_tensor(x).cuda()  # noqa: E731
    a, b = case(50, 9, 3, 30011, torch.bfloat16), case(51, 17, 2, 12345, torch.bfloat16, True)
    graphs = []
    for c in (a, b):
        buf = {k: cuda(c[k]) for k in ("logits", "drafts", "u", "temperature", "draft_logits")}
        run = lambda buf=buf: sampler.spec_verify(buf["logits"], buf["drafts"], buf["u"], buf["temperature"],  # noqa: E731
                                                  draft_logits=buf["draft_logits"])
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            eager = run()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            out = run()
        stream.synchronize()
        graphs.append((g, out, eager, buf, run))
    for g, out, eager, buf, run in graphs + graphs[::-1]:
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out.tokens, eager.tokens) and torch.equal(out.logprob, eager.logprob)
    for g, out, eager, buf, run in graphs:
        buf["u"].copy_(1.0 - buf["u"])
        g.replay()
        again = run()
        torch.cuda.synchronize()
        assert torch.equal(out.tokens, again.tokens) and torch.equal(out.n_kept, again.n_kept)


def test_results_repeat(gpu_sampler_factory):
    c = case(91, 64, 4, 50257)
    outs = [compare(gpu_sampler_factory(129280, 512), c) for _ in range(3)]
    for o in outs[1:]:
        assert torch.equal(o.tokens, outs[0].tokens) and torch.equal(o.logprob, outs[0].logprob)


def test_refusals(gpu_sampler_factory):
    from mako_b200 import BatchSampler, MakoError
    sampler = BatchSampler(100, 4)
    z = lambda *n, t=torch.float32: torch.zeros(*n, dtype=t, device="cuda")  # noqa: E731
    i = lambda *n: z(*n, t=torch.int32)  # noqa: E731
    with pytest.raises(MakoError, match="n_vocab 101"):
        sampler.spec_verify(z(4, 101), i(2, 1), z(2, 3), 1.0)
    with pytest.raises(MakoError, match="n_seq 5"):
        sampler.spec_verify(z(5, 100), i(5, 0), z(5, 2), 1.0)
    with pytest.raises(MakoError, match="mask_ld 3"):
        sampler.spec_verify(z(4, 100), i(2, 1), z(2, 3), 1.0, mask=i(4, 3))
    with pytest.raises(MakoError, match="finite"):
        sampler.spec_verify(z(4, 100), i(2, 1), z(2, 3), math.nan)
    with pytest.raises(AssertionError):
        sampler.spec_verify(z(4, 100), i(2, 1), z(2, 2), 1.0)
    with pytest.raises(AssertionError):
        sampler.spec_verify(z(4, 100), i(2, 1), z(2, 3), 1.0, draft_logits=z(2, 100, t=torch.bfloat16))
    with pytest.raises(KeyError):
        sampler.spec_verify(z(4, 100, t=torch.float64), i(2, 1), z(2, 3), 1.0)
    got = sampler.spec_verify(z(0, 100), i(0, 1), z(0, 3), 1.0)
    assert got.n_kept.numel() == 0
