"""Verification of drafts (mk_spec_verify) where its single-precision sums end and where probabilities are next to nothing or next to
each other, against the 64-bit form."""
import math

import numpy as np
import pytest
import torch

from tests import test_gpu_spec_verify as verify

pytestmark = pytest.mark.gpu


def plain(s, d, v, logits, drafts, u, temperature, draft_logits=None, draft_temperature=None):
    f32 = lambda x: np.asarray(x, np.float32)  # noqa: E731
    c = {"logits": torch.from_numpy(f32(logits).reshape(s * (d + 1), v)), "drafts": np.asarray(drafts, np.int32).reshape(s, d),
         "u": f32(u).reshape(s, d + 2), "temperature": np.broadcast_to(f32(temperature), (s,)).copy(), "mask": None, "mask_drafts": False,
         "draft_logits": None if draft_logits is None else torch.from_numpy(f32(draft_logits).reshape(s * d, v))}
    if draft_temperature is not None:
        c["draft_temperature"] = np.broadcast_to(f32(draft_temperature), (s,)).copy()
    return c


def test_a_part_of_a_row_beyond_the_line(gpu_sampler_factory):
    """Two columns of different threads' on the two sides of 1e6 (693147 log2 e): P is 0.622 and 0.378."""
    row = np.full((2, 40), -np.inf, np.float32)
    row[:, 0], row[:, 16] = -693147.0, -693147.5
    c = plain(1, 1, 40, row, [[0]], [[0.9, 0.3, 0.5]], 1.0)
    got = verify.compare(gpu_sampler_factory(129280, 512), c)
    assert got.n_kept.tolist() == [0] and got.next_token.tolist() == [16]
    c["u"][0] = 0.5
    got = verify.compare(gpu_sampler_factory(129280, 512), c)
    assert got.n_kept.tolist() == [1]


@pytest.mark.parametrize("onehot", [False, True])
@pytest.mark.parametrize("temperature", [1.0, 1e-4])
@pytest.mark.parametrize("v", [61, 5003, 100003])
def test_rows_on_both_sides_of_the_line(gpu_sampler_factory, v, temperature, onehot):
    """Largest logits over T whose log2 lies just inside or just outside of 1e6, of either sign, and at 1e6 + 4096."""
    rng = np.random.default_rng(v)
    tops = [side * (line + off) for line in (1e6, 1e6 + 4096) for side in (-1, 1) for off in (-30.0, -1.0, -0.1, 0.1, 1.0, 30.0)]
    s, t = len(tops), np.float32(temperature)
    base = np.array(tops)[:, None, None] * math.log(2) * float(t)

    def rows(n):
        below = rng.exponential(4.0, (s, n, v)) * (rng.random((s, n, v)) < 0.9)
        return (base - below * float(t)).astype(np.float32)

    target, draft = rows(2), rows(1)
    drafts = np.argmax(draft[:, 0] / t + rng.gumbel(size=(s, v)), axis=1)
    c = plain(s, 1, v, target, drafts, rng.random((s, 3)), t, None if onehot else draft)
    verify.compare(gpu_sampler_factory(129280, 512), c)


@pytest.mark.parametrize("swap", [False, True])
def test_a_residual_between_rows_of_far_temperatures(gpu_sampler_factory, swap):
    """log2(e) / T as fp32 is off by 2^-25 of itself, which at a logit of 9e5 times T is 0.03 of a power of two, up for one of these
    temperatures and down for the other. Eight columns, all alike in P; Q has more on the draft: the draft has no part in the rest."""
    tp, tq = (2.5843542971415445e-05, 2.517000939405989e-05)[::-1 if swap else 1]
    p = np.full((2, 8), 15.0, np.float32)
    q = p[:1].copy()
    q[0, 0] = np.nextafter(np.float32(15), np.float32(16))
    us = [0.002, 0.05, 0.2, 0.4, 0.6, 0.97]
    n = len(us)
    c = plain(n, 1, 8, np.tile(p, (n, 1, 1)), [[0]] * n, [[0.995, x, 0.5] for x in us], tp, np.tile(q, (n, 1, 1)), tq)
    got = verify.compare(gpu_sampler_factory(129280, 512), c)
    assert got.n_kept.tolist() == [0] * n and got.next_token.tolist() == [1 + int(7 * x) for x in us]


def test_probabilities_next_to_nothing(gpu_sampler_factory):
    """P and u Q of 2^-120 to 2^-160, which fp32 holds in few bits or not at all: kept iff u Q is below P, by a tenth or by much."""
    rng = np.random.default_rng(5)
    cases = [(-127.0, -125.0, 2.0 ** -5), (-127.4, -120.0, 2.0 ** -7.3), (-130.0, -133.0, 0.5), (-140.0, -140.0, 0.99)]
    for e in np.arange(-160.0, -100.0, 0.5):
        for by in (0.9, 1.1, 0.5, 2.0):
            u = rng.uniform(0.01, 0.45)
            cases.append((e, e + math.log2(by / u), u))
    s, v = len(cases), 4096
    p, q = np.full((s, 2, v), -np.inf, np.float32), np.full((s, 1, v), -np.inf, np.float32)
    for i, (ep, eq, _) in enumerate(cases):
        n = 1 if i % 2 else v - 1  # what has the rest: one column, or all others
        p[i, :, :n] = q[i, :, :n] = 0.0
        p[i, 0, -1], q[i, 0, -1] = ep * math.log(2), eq * math.log(2)
    u = np.array([[x[2], 0.5, 0.5] for x in cases], np.float32)
    dist = lambda x: np.exp(x[:, 0, -1].astype(np.float64)) / (np.exp(x[:, 0].astype(np.float64)).sum(1))  # noqa: E731
    lhs, rhs = u[:, 0].astype(np.float64) * dist(q), dist(p)
    assert (np.abs(lhs - rhs) > 0.005 * rhs).all()
    cuda = lambda x: torch.from_numpy(x).cuda()  # noqa: E731
    got = gpu_sampler_factory(129280, 512).spec_verify(
        cuda(p.reshape(2 * s, v)), torch.full((s, 1), v - 1, dtype=torch.int32, device="cuda"), cuda(u), 1.0,
        draft_logits=cuda(q.reshape(s, v)))
    assert np.array_equal(got.n_kept.cpu().numpy(), (lhs < rhs).astype(np.int32))


@pytest.mark.parametrize("seed", range(4))
def test_a_residual_of_next_to_nothing(gpu_sampler_factory, seed):
    """P and Q alike to 1e-7 in every column but the draft's, where Q has twice P's 1e-8: the rest is a few 1e-8 of the whole, spread over
    the columns whose part is above the average change."""
    rng = np.random.default_rng(seed)
    s, v = 40, 1000
    q = np.zeros((s, 1, v), np.float32)
    p = np.concatenate([rng.uniform(0.0, 1e-7, (s, 1, v)), np.zeros((s, 1, v))], 1).astype(np.float32)
    p[:, 0, 7], q[:, 0, 7] = math.log(1e-5), math.log(2e-5)
    c = plain(s, 1, v, p, np.full((s, 1), 7), np.stack([np.full(s, 0.9), rng.random(s), rng.random(s)], 1), 1.0, q)
    verify.compare(gpu_sampler_factory(129280, 512), c)


def test_temperatures_whose_inverse_passes_fp32(gpu_sampler_factory):
    """log2(e) / T above fp32's range, and logits of that temperature's size: P is 0.622 and 0.378."""
    row = np.full((2, 40), -1.0, np.float32)
    row[:, 0], row[:, 16] = 0.0, -1e-39
    c = plain(2, 1, 40, np.tile(row, (2, 1, 1)), [[0], [0]], [[0.9, 0.3, 0.5], [0.5, 0.3, 0.7]], 2e-39)
    got = verify.compare(gpu_sampler_factory(129280, 512), c)
    # the second one keeps its draft; the token behind it is drawn with 0.3, which is below 0.622
    assert got.n_kept.tolist() == [0, 1] and got.next_token.tolist() == [16, 0]


def test_p_and_q_alike_but_for_what_is_next_to_nothing(gpu_sampler_factory):
    """Both rows are one token's, all but 2e-28 of P and less of Q, and the draft weighs nothing in either: what P has above Q is spread over
    the others, however little it is; 1 - 1 is nothing."""
    v, n = 500, 24
    rng = np.random.default_rng(3)
    p, q = np.full((n, 2, v), -np.inf, np.float32), np.full((n, 1, v), -np.inf, np.float32)
    p[:, :, 33], q[:, :, 33] = rng.uniform(0.2, 0.5, (n, 1)), rng.uniform(0.2, 0.5, (n, 1))
    p[:, :, 17], q[:, :, 17] = p[:, :, 33] - 0.085, q[:, :, 33] - 0.2
    p[:, :, 400], q[:, :, 400] = p[:, :, 33] - 0.0855, q[:, :, 33] - 0.2
    c = plain(n, 1, v, p, np.full((n, 1), 5), np.stack([np.full(n, 0.5), rng.random(n), rng.random(n)], 1), 0.00135, q)
    got = verify.compare(gpu_sampler_factory(129280, 512), c)
    assert set(got.next_token.tolist()) == {17, 400}


def test_p_and_q_the_same_but_for_a_constant(gpu_sampler_factory):
    """A draft that weighs nothing in either is refused; max(0, P - Q) is nothing, so P is drawn from (in 64 bits P - Q is of roundings)."""
    v, n = 1000, 200
    rng = np.random.default_rng(4)
    p = np.round(rng.normal(0.0, 2.0, (n, 2, v)) * 1024) / 1024
    p[:, :, 5] = -np.inf
    q = p[:, :1] + rng.integers(1, 2048, (n, 1, 1)) / 512
    u = np.stack([np.full(n, 0.5), rng.random(n), rng.random(n)], 1).astype(np.float32)
    c = plain(n, 1, v, p, np.full((n, 1), 5), u, 0.7, q)
    cuda = lambda x: torch.as_tensor(x).cuda()  # noqa: E731
    got = gpu_sampler_factory(129280, 512).spec_verify(cuda(c["logits"]), cuda(c["drafts"]), cuda(c["u"]), cuda(c["temperature"]),
                                                       draft_logits=cuda(c["draft_logits"]))
    run = np.cumsum(np.exp(p[:, 0] / float(np.float32(0.7))), 1)
    want = (run <= u[:, 1:2].astype(np.float64) * run[:, -1:]).sum(1)
    assert got.n_kept.tolist() == [0] * n and got.next_token.tolist() == want.tolist()
