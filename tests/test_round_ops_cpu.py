"""CPU tests of the serving round's operators: what their entry points refuse before any device is touched, and the plain forms
that the GPU tests compare with, on answers that are known."""
import ctypes as C

import numpy as np
import torch

from tests import round_oracle as oracle


def test_null_handles_are_refused():
    from mako_b200._lib import HeadC, KvPagesC, KvPlanC, SpecRowsC, lib
    assert lib.mk_head_logits(None, C.byref(HeadC()), None, 0, None, 0, None, 0, None) == 1
    assert lib.mk_spec_verify(None, C.byref(SpecRowsC()), None, None, None, None, None, None) == 1
    assert lib.mk_kv_plan_step(None, C.byref(KvPagesC()), None, None, 0, C.byref(KvPlanC()), None) == 1
    assert b"mk_kv_plan_step" in lib.mk_last_error()


def test_plan_takes_from_the_top_and_gives_back_first_on_top():
    table = np.array([[4, -1, -1], [5, 6, 7], [-1, -1, -1]], np.int32)
    out, (t, held, free, n) = oracle.plan(table, np.array([1, 3, 0], np.int32), np.array([1, 2, 3, -1, -1, -1], np.int32), 3,
                                          [3, 0, 0], [4, 0, 1], 4, 8)
    # sequence 1 gives 5 6 7 back, 5 topmost; sequence 0 takes 5, sequence 2 takes 6
    assert t.tolist() == [[4, 5, -1], [-1, -1, -1], [6, -1, -1]] and held.tolist() == [2, 0, 1]
    assert n == 4 and free[:4].tolist() == [1, 2, 3, 7]
    assert out["query_start"] == [0, 4, 4, 5] and out["positions"] == [3, 4, 5, 6, 0, 0, 0, 0]
    assert out["slots"] == [19, 20, 21, 22, 24, -1, -1, -1] and out["token_seq"] == [0, 0, 0, 0, 2, -1, -1, -1]


def test_plan_keeps_every_page_once():
    rng = np.random.default_rng(0)
    s, cols, total = 30, 12, 200
    table, held, free, n = np.full((s, cols), -1, np.int32), np.zeros(s, np.int32), np.arange(total, dtype=np.int32), total
    for _ in range(50):
        out, (table, held, free, n) = oracle.plan(table, held, free, n, rng.integers(0, 60, s), rng.integers(0, 20, s), 8, 200)
        pages = np.concatenate([table[i, :held[i]] for i in range(s)] + [free[:n]])
        assert np.array_equal(np.sort(pages), np.arange(total))
        real = [x for x in out["slots"] if x >= 0]
        assert len(set(real)) == len(real)


def test_verify_yields_the_targets_distribution():
    """Over a grid of the uniforms, what a round yields first is spread as the target's softmax."""
    p, q = np.log(np.array([0.5, 0.3, 0.2])), np.log(np.array([0.2, 0.2, 0.6]))
    mass = np.zeros(3)
    grid = (np.arange(40) + 0.5) / 40
    for d, share in enumerate((0.2, 0.2, 0.6)):
        for u0 in grid:
            for u1 in grid:
                _, _, tokens, *_ = oracle.verify(np.stack([p, p]), np.array([[d]], np.int32), np.array([[u0, u1, 0.5]]), [1.0], q[None])[0]
                mass[tokens[0]] += share / 1600
    assert np.allclose(mass, [0.5, 0.3, 0.2], atol=0.02)


def test_head_oracle_is_the_product():
    g = torch.Generator().manual_seed(0)
    h, w, d, u = (torch.randn(*s, generator=g).double() for s in ((3, 8), (5, 8), (2, 4, 8), (2, 5, 4)))
    got, bound = oracle.head(h.numpy(), w.numpy(), np.array([1, -1, 0]), d.numpy(), u.numpy(), np.array([2.0, 3.0]))
    full = torch.stack([w + 3 * u[1] @ d[1], w, w + 2 * u[0] @ d[0]])
    assert np.allclose(got, torch.einsum("tvk,tk->tv", full, h).numpy(), rtol=1e-12) and (bound > 0).all()
