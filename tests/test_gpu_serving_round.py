"""The operators of a serving round one behind the other, as a server runs them: hidden states to logits, the verification of
the drafts, their commit, the pages of the next pass; and all of it captured into one graph, for several rounds."""
import numpy as np
import pytest
import torch

from tests import round_oracle as oracle

pytestmark = pytest.mark.gpu


def test_rounds_in_one_graph():
    from mako_b200 import BatchSampler, KvPlan
    rng = np.random.default_rng(4)
    s, d, v, dim, rank, n, page = 12, 3, 2003, 128, 16, 5, 4
    n_pos, cap, cols = d + 1, 64, 40
    sampler = BatchSampler(v, s * n_pos)
    f = lambda *k, t=torch.bfloat16: torch.from_numpy(rng.normal(size=k).astype(np.float32)).cuda().to(t)  # noqa: E731
    i32 = lambda x: torch.as_tensor(np.asarray(x, np.int32)).cuda()  # noqa: E731
    weight, down, up, scale = f(v, dim) * 0.3, f(n, rank, dim) * 0.1, f(n, v, rank) * 0.3, f(n, t=torch.float32).abs()
    adapter = i32(np.repeat(rng.integers(-1, n, s), n_pos))
    hidden, draft_logits, drafts = f(s * n_pos, dim), f(s * d, v, t=torch.float32), i32(rng.integers(0, v, (s, d)))
    u = torch.rand(s, n_pos + 1, device="cuda")
    history, length = torch.zeros(s, cap, dtype=torch.int32, device="cuda"), i32(rng.integers(1, 9, s))
    held0 = -(-length.cpu().numpy() // page)
    table = np.full((s, cols), -1, np.int32)
    ids = rng.permutation(s * cols).astype(np.int32)
    at = 0
    for k in range(s):
        table[k, :held0[k]] = ids[at:at + held0[k]]
        at += held0[k]
    free = np.concatenate([ids[at:], np.full(at, -1, np.int32)])
    pages = [i32(table), i32(held0), i32(free), i32([len(ids) - at])]
    fresh, plan = i32([n_pos] * s), KvPlan.empty(s, s * n_pos + 3)
    logits, nxt = torch.empty(s * n_pos, v, device="cuda"), i32([0] * s)

    def step():
        sampler.head_logits(hidden, weight, adapter=adapter, down=down, up=up, scale=scale, out=logits)
        r = sampler.spec_verify(logits, drafts, u, 0.9, draft_logits=draft_logits)
        sampler.spec_commit(drafts, r.n_kept, r.next_token, history, length, next_input=nxt)
        sampler.kv_plan(*pages, length, fresh, page_size=page, out=plan)
        return r

    start = [x.clone() for x in pages + [history, length]]
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        step()
    stream.synchronize()
    for x, y in zip(pages + [history, length], start):
        x.copy_(y)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=stream):
        r = step()
    state = (table, held0.astype(np.int32), free, len(ids) - at)
    want_len, want_hist = length.cpu().numpy().copy(), history.cpu().numpy().copy()
    for turn in range(3):
        hidden.copy_(f(s * n_pos, dim))
        u.copy_(torch.from_numpy(rng.random((s, n_pos + 1)).astype(np.float32)))
        drafts.copy_(i32(rng.integers(0, v, (s, d))))
        exact, bound = oracle.head(*(x.double().cpu().numpy() for x in (hidden, weight)), adapter.cpu().numpy(),
                                   *(x.double().cpu().numpy() for x in (down, up, scale)))
        for k in range(s):  # a draft that both sides like, now and then
            draft_logits.view(s, d, v)[k, 0, int(drafts[k, 0])] = 12.0 if turn else 9.0
            hidden.view(s, n_pos, dim)[k, 0] = 4.0 * weight[int(drafts[k, 0])].to(hidden.dtype) if k % 2 else hidden.view(s, n_pos, dim)[k, 0]
        exact, bound = oracle.head(*(x.double().cpu().numpy() for x in (hidden, weight)), adapter.cpu().numpy(),
                                   *(x.double().cpu().numpy() for x in (down, up, scale)))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert (np.abs(logits.double().cpu().numpy() - exact) <= bound).all()
        rounds = oracle.verify(logits.double().cpu().numpy(), drafts.cpu().numpy(), u.cpu().numpy(), np.full(s, np.float32(0.9)),
                               draft_logits.double().cpu().numpy())
        assert r.n_kept.tolist() == [x[0] for x in rounds] and r.next_token.tolist() == [x[1] for x in rounds]
        for k, (kept, token, *_) in enumerate(rounds):
            new = drafts.cpu().numpy()[k, :kept].tolist() + [token]
            want_hist[k, want_len[k]:want_len[k] + len(new)] = new
            want_len[k] += len(new)
        assert np.array_equal(length.cpu().numpy(), want_len) and np.array_equal(history.cpu().numpy(), want_hist)
        want, state = oracle.plan(*state, want_len, [n_pos] * s, page, s * n_pos + 3)
        for key, x in want.items():
            assert np.array_equal(getattr(plan, key).cpu().numpy().astype(np.int64), np.asarray(x, dtype=np.int64)), key
    assert any(k for k in r.n_kept.tolist())
