"""A server's passes with the cache: pages planned, keys and values appended with their rotation, attention over the cache, the head, and the
sampled tokens' log-probabilities, captured once for passes of mixed lengths and replayed; a speculative round that takes tokens back."""
import math

import numpy as np
import pytest
import torch

from tests import kv_oracle as oracle

pytestmark = pytest.mark.gpu


def test_passes_in_one_graph():
    from mako_b200 import BatchSampler, KvCache, KvPlan, SamplingParams
    rng = np.random.default_rng(5)
    s, heads, q_heads, dim, page, v, most = 6, 2, 8, 64, 16, 1009, 120
    sampler = BatchSampler(v, s)
    pages, cols = 60, 20
    i32 = lambda x: torch.as_tensor(np.asarray(x, np.int32)).cuda()  # noqa: E731
    table, held, free, n_free = i32(np.full((s, cols), -1)), i32([0] * s), i32(rng.permutation(pages)), i32([pages])
    length, fresh = i32([0] * s), i32([0] * s)
    cache, plan = KvCache.empty(pages, heads, page, dim), KvPlan.empty(s, most)
    qkv = torch.zeros(most, q_heads + 2 * heads, dim, device="cuda").bfloat16()
    freq = torch.from_numpy((10000.0 ** (-np.arange(dim // 2) * 2.0 / dim)).astype(np.float32)).cuda()
    weight = torch.from_numpy(rng.normal(0, 0.05, (v, q_heads * dim)).astype(np.float32)).cuda().bfloat16()
    last, u, tokens = torch.zeros(s, dtype=torch.int64, device="cuda"), torch.zeros(s, device="cuda"), torch.zeros(s, dtype=torch.int32, device="cuda")
    q, k, values = qkv.split([q_heads, heads, heads], 1)
    rotated, out = torch.zeros_like(q.contiguous()), torch.zeros(most, q_heads, dim, device="cuda").bfloat16()
    params = SamplingParams(temperature=0.9)

    def step():
        sampler.kv_plan(table, held, free, n_free, length, fresh, page_size=page, out=plan)
        sampler.kv_append(cache, k, values, plan.slots, q=q, q_out=rotated, positions=plan.positions, inv_freq=freq)
        sampler.kv_attention(rotated, cache, table, plan.query_start, plan.kv_len, out=out)
        logits = sampler.head_logits(out.view(most, -1)[last], weight)
        tokens.copy_(sampler.sample(logits, params, u).token)
        return logits, sampler.token_logprobs(logits, tokens, 0.9, top=4)

    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        step()
    stream.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=stream):
        logits, logprobs = step()
    lengths = np.zeros(s, np.int64)
    # prompts, then tokens one by one with a prompt beside them, a speculative round, its drafts taken back, a sequence that ends
    for new, back in (([40, 7, 0, 33, 1, 16], None), ([1, 1, 50, 1, 1, 1], None), ([4, 4, 4, 4, 4, 4], [1, 4, 0, 2, 3, 4]), ([1, 1, 1, 0, 1, 1], None)):
        for t in (qkv, u):
            t.copy_(torch.from_numpy((rng.normal(0, 1, t.shape) if t is qkv else rng.random(t.shape)).astype(np.float32)))
        length.copy_(i32(lengths))
        fresh.copy_(i32(new))
        starts = np.concatenate([[0], np.cumsum(new)])
        last.copy_(torch.from_numpy(np.maximum(starts[1:] - 1, 0)))
        k0, ks0 = cache.k.double().cpu().numpy(), cache.k_scale.double().cpu().numpy()
        v0, vs0 = cache.v.double().cpu().numpy(), cache.v_scale.double().cpu().numpy()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        slots, positions = plan.slots.cpu().numpy(), plan.positions.cpu().numpy()
        assert plan.flags.tolist() == [0] * s and plan.kv_len.tolist() == (lengths + new).tolist()
        x = qkv.double().cpu().numpy()
        # values exactly; keys and queries by what attention makes of them, from the codes that are there and the rotated queries
        oracle.append(v0, vs0, x[:, q_heads + heads:], slots, page)
        assert np.array_equal(cache.v.double().cpu().numpy(), v0) and np.array_equal(cache.v_scale.double().cpu().numpy(), vs0)
        turned = np.stack([oracle.rotate(x[i, :q_heads + heads], float(positions[i]), freq.double().cpu().numpy(), False, 1.0)[0] for i in range(most)])
        oracle.append(k0, ks0, turned[:, q_heads:], slots, page)
        got = cache.k.double().cpu().numpy() * cache.k_scale.double().cpu().numpy()[:, :, None, None]
        real = slots >= 0
        for i in np.flatnonzero(real):
            p, at = slots[i] // page, slots[i] % page
            step_of = np.maximum(np.abs(turned[i, q_heads:]) * 2.0 ** -4, ks0[p][:, None] * 2.0 ** -10)
            assert (np.abs(got[p, :, at] - turned[i, q_heads:]) <= step_of * (1 + 2.0 ** -8) + 1e-5).all()
        wide = lambda y, z: y.float().cpu().double() * z.double().cpu().view(*z.shape, 1, 1)  # noqa: E731
        want, bound = oracle.attention(rotated.double().cpu(), wide(cache.k, cache.k_scale), wide(cache.v, cache.v_scale), table.cpu().numpy(),
                                       starts, lengths + new, page, 1 / math.sqrt(dim), 0, torch.bfloat16)
        for t, y in want.items():
            assert ((out[t].double().cpu() - y).abs() <= bound[t]).all(), t
        rows = logits.double().cpu().numpy()
        for i in range(s):
            lp, _, ids, tops, room, _ = oracle.logprobs(rows[i], [int(tokens[i])], float(np.float32(0.9)), 4)
            assert logprobs.top_ids[i].tolist() == ids.tolist()
            assert abs(float(logprobs.logprob[i]) - lp[0]) <= room[int(tokens[i])]
        lengths = lengths + (new if back is None else back)


def test_appends_are_seen_by_the_next_attention_of_the_stream():
    """The token of a step attends to itself: its key and value are in the cache when the queries are read."""
    from mako_b200 import BatchSampler, KvCache
    sampler = BatchSampler(32, 1)
    cache = KvCache.empty(4, 1, 16, 64)
    x = torch.randn(1, 3, 64, device="cuda").half()
    sampler.kv_append(cache, x[:, 1:2], x[:, 2:], torch.tensor([35], device="cuda"))
    # one key: its value, as 8 bits have it
    i32 = lambda *y: torch.tensor(y, dtype=torch.int32, device="cuda")  # noqa: E731
    out = sampler.kv_attention(x[:, :1], KvCache(cache.k[2:3, :, 3:4], cache.v[2:3, :, 3:4], cache.k_scale[2:3], cache.v_scale[2:3]), i32(0).view(1, 1), i32(0, 1),
                               i32(1), max_new=1)
    want = cache.v[2, :, 3].float() * cache.v_scale[2].view(1, 1)
    assert torch.equal(out.float(), want.view(1, 1, 64))
