"""Block tables and slot maps built on the device (mk_kv_plan_step) against a host that serves the sequences one by one."""
import numpy as np
import pytest
import torch

from tests import round_oracle as oracle

pytestmark = pytest.mark.gpu


def make(rng, s, page, longest, new, spare, cols=None):
    ln = rng.integers(0, longest + 1, s).astype(np.int32)
    nw = rng.integers(0, new + 1, s).astype(np.int32)
    need = -(-(longest + new) // page)
    cols = cols or need + 1
    held = (-(-ln // page) + rng.integers(-1, 2, s)).clip(0, cols).astype(np.int32)
    n = int(held.sum())
    ids = rng.permutation(n + spare).astype(np.int32)
    table = np.full((s, cols), -1, np.int32)
    at = 0
    for i in range(s):
        table[i, :held[i]] = ids[at:at + held[i]]
        at += held[i]
    free = np.full(n + spare, -1, np.int32)
    free[:spare] = ids[n:]
    return table, held, free, spare, ln, nw


def both(factory, table, held, free, n_free, ln, nw, page, max_tokens, ld=None):
    from mako_b200 import KvPlan
    s = table.shape[0]
    want, left = oracle.plan(table, held, free, n_free, ln, nw if nw is not None else [0] * s, page, max_tokens)
    sampler = factory(32, 1)
    wide = torch.full((s, ld or table.shape[1]), -7, dtype=torch.int32)
    wide[:, :table.shape[1]] = torch.from_numpy(table)
    d_wide = wide.cuda()
    d_table = d_wide[:, :table.shape[1]]
    d = [torch.from_numpy(np.asarray(x, dtype=np.int32)).cuda() for x in (held, free, np.array([n_free]), ln)]
    plan = KvPlan.empty(s, max_tokens)
    got = sampler.kv_plan(d_table, *d, torch.from_numpy(nw).cuda() if nw is not None else None, page_size=page, out=plan)
    for k, x in want.items():
        assert np.array_equal(getattr(got, k).cpu().numpy().astype(np.int64), np.asarray(x, dtype=np.int64)), k
    assert np.array_equal(d_table.cpu().numpy(), left[0])
    assert (d_wide[:, table.shape[1]:] == -7).all()
    assert np.array_equal(d[0].cpu().numpy(), left[1])
    assert int(d[2]) == left[3]
    assert np.array_equal(d[1].cpu().numpy()[:left[3]], left[2][:left[3]])
    return got


@pytest.mark.parametrize("seed, s, page, longest, new, spare, max_tokens, ld", [
    (1, 1, 16, 40, 1, 4, 1, None), (2, 1, 1, 5, 3, 8, 16, None), (3, 33, 16, 300, 8, 200, 400, None),
    (4, 1000, 32, 900, 8, 2000, 8000, 64), (5, 1025, 16, 100, 3, 3000, 4000, None), (6, 2500, 24, 65, 2, 9000, 5500, None),
    (7, 64, 64, 70000, 4096, 10000, 64 * 4096, None), (8, 7, 7, 50, 200, 400, 1400, 90), (9, 40, 16, 0, 5, 100, 200, None),
    (10, 3, 4096, 9000, 5, 9, 20, None), (11, 148, 16, 4000, 1, 300, 148, None)])
def test_against_the_host(gpu_sampler_factory, seed, s, page, longest, new, spare, max_tokens, ld):
    rng = np.random.default_rng(seed)
    case = make(rng, s, page, longest, new, spare)
    both(gpu_sampler_factory, *case, page, max_tokens, ld)


@pytest.mark.parametrize("seed", range(6))
def test_too_few_pages_or_places(gpu_sampler_factory, seed):
    """Sequences are refused in order, invalid ones in between are left alone, and what is refused keeps what it has."""
    rng = np.random.default_rng(100 + seed)
    table, held, free, n_free, ln, nw = make(rng, 200 if seed % 2 else 1500, 16, 500, 40, 60 + 300 * (seed % 3))
    ln[::17], nw[5::23] = -3, -1
    held[9::31] = table.shape[1] + 1
    ln[13::37] = 2 ** 31 - 1
    both(gpu_sampler_factory, table, held, free, n_free, ln, nw, 16, int(nw.clip(0).sum()) - 200 * (seed % 2))


def test_nothing_fits(gpu_sampler_factory):
    rng = np.random.default_rng(5)
    table, held, free, n_free, ln, nw = make(rng, 50, 16, 100, 4, 0)
    both(gpu_sampler_factory, table, held, free, n_free, ln, nw, 16, 0)
    both(gpu_sampler_factory, table, held, free[:0], 0, ln, nw, 16, 100)  # no room on the list: nothing is given back
    both(gpu_sampler_factory, table, held, free, -5, ln, nw, 16, 100)


def test_no_sequences(gpu_sampler_factory):
    from mako_b200 import KvPlan
    e = lambda *n: torch.zeros(*n, dtype=torch.int32, device="cuda")  # noqa: E731
    plan = gpu_sampler_factory(32, 1).kv_plan(e(0, 4), e(0), e(8), e(1), e(0), e(0), page_size=16, out=KvPlan.empty(0, 9))
    assert int(plan.query_start[0]) == 0 and (plan.slots == -1).all() and (plan.token_seq == -1).all()


def test_finished_sequences_give_all_back_and_pages_come_again(gpu_sampler_factory):
    """Taken and given back, the list is what it was; and without outputs nothing but the pages changes."""
    from mako_b200 import KvPlan
    rng = np.random.default_rng(8)
    table, held, free, n_free, ln, nw = make(rng, 300, 16, 200, 30, 2000)
    held = (-(-ln // 16)).astype(np.int32)
    n = int(held.sum())
    ids = rng.permutation(n + 2000).astype(np.int32)
    table[:] = -1
    for i, at in enumerate(np.cumsum(held) - held):
        table[i, :held[i]] = ids[at:at + held[i]]
    free = np.concatenate([ids[n:], np.full(n, -1, np.int32)])
    d = [torch.from_numpy(x.copy()).cuda() for x in (table, held, free, np.array([2000], np.int32), ln)]
    sampler = gpu_sampler_factory(32, 1)
    sampler.kv_plan(*d, torch.from_numpy(nw).cuda(), page_size=16, out=KvPlan.empty(300, 9000))
    assert int(d[3]) < 2000
    sampler.kv_plan(*d, page_size=16)
    for x, y in zip(d, (table, held, free, np.array([2000], np.int32), ln)):
        assert np.array_equal(x.cpu().numpy(), y)
    d[4].zero_()
    sampler.kv_plan(*d, page_size=16)
    assert int(d[3]) == n + 2000 and (d[0] == -1).all() and (d[1] == 0).all()
    assert np.array_equal(np.sort(d[2].cpu().numpy()), np.arange(n + 2000))


def test_slots_pass_32_bits(gpu_sampler_factory):
    table = np.array([[2_000_000_000, 7]], np.int32)
    got = both(gpu_sampler_factory, table, np.array([2], np.int32), np.zeros(1, np.int32), 0, np.array([14], np.int32),
               np.array([5], np.int32), 16, 6)
    assert int(got.slots[0]) == 2_000_000_000 * 16 + 14


def test_captured_with_a_loop_of_rounds(gpu_sampler_factory):
    """A captured plan follows the lengths that the device holds, round after round."""
    from mako_b200 import KvPlan
    rng = np.random.default_rng(21)
    sampler = gpu_sampler_factory(32, 1)
    table, held, free, n_free, ln, nw = make(rng, 40, 16, 60, 5, 600)
    table = np.pad(table, ((0, 0), (0, 20)), constant_values=-1)
    d = [torch.from_numpy(np.asarray(x, np.int32)).cuda() for x in (table, held, free, np.array([n_free]), ln)]
    d_new, plan = torch.from_numpy(nw).cuda(), KvPlan.empty(40, 256)
    stream = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=stream):
        sampler.kv_plan(*d, d_new, page_size=16, out=plan)
    state = (table, held, free, n_free)
    for _ in range(12):
        g.replay()
        want, state = oracle.plan(*state, ln, nw, 16, 256)
        torch.cuda.synchronize()
        for k, x in want.items():
            assert np.array_equal(getattr(plan, k).cpu().numpy().astype(np.int64), np.asarray(x, dtype=np.int64)), k
        ln = np.asarray(want["kv_len"], np.int32) - rng.integers(0, 3, 40).clip(0, np.asarray(want["kv_len"])).astype(np.int32)
        nw = rng.integers(0, 6, 40).astype(np.int32)
        ln[rng.integers(0, 40)] = 0
        d[4].copy_(torch.from_numpy(ln))
        d_new.copy_(torch.from_numpy(nw))
        torch.cuda.synchronize()


def test_refusals(gpu_sampler_factory):
    from mako_b200 import MakoError
    sampler = gpu_sampler_factory(32, 1)
    e = lambda *n: torch.zeros(*n, dtype=torch.int32, device="cuda")  # noqa: E731
    with pytest.raises(MakoError, match="page_size 0"):
        sampler.kv_plan(e(2, 4), e(2), e(8), e(1), e(2), page_size=0)
    with pytest.raises(AssertionError):
        sampler.kv_plan(e(2, 4), e(3), e(8), e(1), e(2), page_size=16)
    with pytest.raises(AssertionError):
        sampler.kv_plan(e(2, 4), e(2), e(8), e(1), e(2), e(2), page_size=16)  # tokens, and nowhere to write them
