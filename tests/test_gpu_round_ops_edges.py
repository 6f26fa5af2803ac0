"""The serving round's operators where sizes, values and neighbours are unusual: long rounds, wide vocabularies, logits and
temperatures far from one, many rows, several handles at once."""
import math

import numpy as np
import pytest
import torch

from tests import test_gpu_head_logits as head
from tests import test_gpu_spec_verify as verify

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("s, d, v", [(3, 40, 700), (2, 70, 129), (1, 33, 5000)])
def test_rounds_of_many_drafts(gpu_sampler_factory, s, d, v):
    """More positions than a warp has lanes, nearly all of them kept."""
    c = verify.case(d, s, d, v, torch.float32, noise=0.05, ragged=False)
    verify.compare(gpu_sampler_factory(129280, 512), c)
    c["draft_logits"] = c["logits"].view(s, d + 1, v)[:, :d].reshape(s * d, v).clone()  # the target's own: all kept
    got = verify.compare(gpu_sampler_factory(129280, 512), c)
    assert got.n_kept.tolist() == [d] * s


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_wide_vocabulary(dtype):
    from mako_b200 import BatchSampler
    sampler = BatchSampler(600011, 3)
    verify.compare(sampler, verify.case(1, 3, 2, 600011, dtype))
    verify.compare(sampler, verify.case(2, 2, 1, 600011, dtype, True, mask=0.01))


def test_logits_and_temperatures_far_from_one(gpu_sampler_factory):
    """Rows whose largest logit times log2(e) / T is beyond the fp32 sums: weighed in 64 bits from the start."""
    sampler = gpu_sampler_factory(129280, 512)
    for seed, scale in ((1, 1e7), (2, 1e20), (3, 3e36)):
        c = verify.case(seed, 8, 2, 2003, torch.float32, ragged=False)
        c["logits"] *= scale / 16
        c["draft_logits"] *= scale / 16
        c["temperature"][:] = (c["temperature"].astype(np.float64) * min(scale, 1e28) / 16).astype(np.float32)
        c["temperature"][::2] = 1.0
        verify.compare(sampler, c)
    c = verify.case(5, 8, 2, 2003, torch.bfloat16, ragged=False)
    c["temperature"][:] = [1e-6, 1e-7, 1e-4, 1e-3, 1e-5, 3e-6, 1e-9, 1e-30]
    verify.compare(sampler, c)
    # whole rows of the type's lowest value: every token as likely as the other
    c = verify.case(6, 6, 1, 999, torch.float32, ragged=False)
    c["logits"].fill_(torch.finfo(torch.float32).min)
    c["draft_logits"][::2] = torch.finfo(torch.float32).min
    verify.compare(sampler, c)


def test_temperatures_that_are_none(gpu_sampler_factory):
    c = verify.case(7, 6, 2, 3000, torch.float32)
    c["temperature"][:] = [math.nan, math.inf, -math.inf, 1e30, 2e-39, 0.7]
    verify.compare(gpu_sampler_factory(129280, 512), c)


@pytest.mark.parametrize("rows, v, dim, rank, n", [(1300, 300, 64, 16, 7), (700, 257, 200, 24, 300), (321, 1000, 128, 128, 3)])
def test_many_rows(rows, v, dim, rank, n):
    """Row tiles of several rounds, and more adapters than a tile has rows."""
    from mako_b200 import BatchSampler
    head.compare(BatchSampler(max(v, 512), rows), head.make(rows, rows, v, dim, rank, n, torch.bfloat16))


def test_handles_side_by_side():
    """Each handle on a stream of its own, all at once, against the same calls one by one."""
    from mako_b200 import BatchSampler
    work = []
    for i in range(4):
        c = {k: x.cuda() for k, x in head.make(60 + i, 20 + 30 * i, 9000, 512, 16, 4, torch.bfloat16).items()}
        h = BatchSampler(9000, 128)
        w = verify.case(70 + i, 12 + 9 * i, 3, 9000, torch.float16)
        w = [torch.as_tensor(w[k]).cuda() for k in ("logits", "drafts", "u", "temperature", "draft_logits")]
        work.append((h, c, w, torch.cuda.Stream()))
    run = lambda h, c, w: (h.head_logits(**c), h.spec_verify(*w[:4], draft_logits=w[4]))  # noqa: E731
    want = [run(*x[:3]) for x in work]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for h, c, w, stream in work:
            with torch.cuda.stream(stream):
                got.append(run(h, c, w))
        torch.cuda.synchronize()
        for (a, b), (x, y) in zip(got, want):
            assert torch.equal(a, x) and torch.equal(b.tokens, y.tokens) and torch.equal(b.logprob, y.logprob)


def test_a_handle_after_its_neighbours_calls(gpu_sampler_factory):
    """Sampling and the round's operators share a handle's memory: one after the other they leave each other's results alone."""
    from mako_b200 import BatchSampler, SamplingParams
    h = BatchSampler(9000, 64)
    g = torch.Generator(device="cuda").manual_seed(3)
    logits, u = torch.randn(40, 9000, device="cuda", generator=g) * 2, torch.rand(40, device="cuda", generator=g)
    p = SamplingParams(temperature=0.9, top_p=0.95)
    c = {k: x.cuda() for k, x in head.make(9, 40, 9000, 256, 32, 5, torch.bfloat16).items()}
    first, second = h.sample(logits, p, u).token.clone(), h.head_logits(**c)
    for _ in range(3):
        assert torch.equal(h.sample(logits, p, u).token, first)
        assert torch.equal(h.head_logits(**c), second)


@pytest.mark.parametrize("rows", [9, 25, 47, 64, 81, 112, 145, 160, 161, 192, 225, 256, 310])
def test_heads_of_several_tiles_a_share(rows):
    """Every number of vocabulary tiles and rows that a thread has, with shares of the vocabulary that fill no number of them."""
    from mako_b200 import BatchSampler
    head.compare(BatchSampler(60007, 512), head.make(rows, rows, 60007, 136, 40, 6, torch.bfloat16))


@pytest.mark.parametrize("rows", [48, 130, 230])
def test_an_adapters_infinities_stay_its_own(gpu_sampler_factory, rows):
    c = head.make(11, rows, 1500, 128, 24, 5, torch.bfloat16)
    sampler = gpu_sampler_factory(129280, 512)
    gpu = {k: x.cuda() for k, x in c.items()}
    call = lambda: sampler.head_logits(gpu["hidden"], gpu["weight"], **{k: gpu[k] for k in ("adapter", "down", "up", "scale")}).cpu()  # noqa: E731
    before = call().clone()
    gpu["up"][2, 700:1100:100] = math.inf
    gpu["up"][2, 900] = math.nan
    after = call()
    hit = torch.zeros(rows, 1500, dtype=torch.bool)
    hit[(c["adapter"] == 2).nonzero(), torch.arange(700, 1100, 100)] = True
    assert hit.any() and not after[hit].isfinite().any()
    assert torch.equal(after[~hit], before[~hit])
