"""64-bit restatements of the operators around the paged cache and of the log-probabilities, on the CPU, with bounds of the kernels' roundings."""
import math

import numpy as np
import torch

E4M3 = torch.float8_e4m3fn


def half_ulp(t):
    return torch.finfo(t).eps / 2


# ---- log-probabilities -----------------------------------------------------------------------------------------------------------

def logprobs(x, tokens, temperature, top, allowed=None):
    """One row, float64: (log-probabilities of the tokens, entropy, ids and log-probabilities of the likeliest, bounds of the two kinds
    of numbers). What a kernel may be off by: a weight's exponent is one rounding of c x - shift (c two roundings from 1 / T) and the
    special-function unit's 2^-22, sums of up to V / 1024 + 64 terms a thread in fp32, a logarithm of two roundings."""
    x = np.asarray(x, np.float64)
    v = len(x)
    live = ~np.isnan(x) & (x > -np.inf)
    if allowed is not None:
        live &= allowed
    order = np.lexsort((np.arange(v), -np.where(live, x, -np.inf)))
    order = order[live[order]]
    lp = np.full(v, -np.inf)
    h, spread, log_s = 0.0, 0.0, 0.0
    if len(order):
        first = order[0]
        if not (1e-30 < temperature < 1e30) or np.isinf(x[first]):
            lp[first] = 0.0
            order = order[:1]
        else:
            y = (x[live] - x[first]) / temperature
            log_s = np.log(np.exp(y).sum())
            lp[live] = y - log_s
            p = np.exp(lp[live])
            h, spread = -(p * lp[live])[p > 0].sum(), -(p * y)[p > 0].sum()
    ids = np.full(top, -1)
    ids[:min(top, len(order))] = order[:top]
    given = np.array([lp[t] if 0 <= t < v else 0.0 for t in tokens])
    chain = (v / 1024 + 64) * 2.0 ** -24 + 2.0 ** -21
    finite = np.where(np.isinf(lp), 0.0, lp)
    bound = 2.0 ** -22 * (np.abs(finite) + 2 * log_s + 1) + chain * (1 + spread)
    return given, h, ids, np.where(ids >= 0, lp[ids], -np.inf), bound, 2.0 ** -21 * (1 + log_s + spread) + 2 * chain * (1 + spread)


# ---- the cache -------------------------------------------------------------------------------------------------------------------

def scale_for(most):
    """The least power of two s with most <= 448 s, at least 2^-100."""
    if most == 0:
        return 2.0 ** -100
    m, e = math.frexp(most / 448.0)
    return 2.0 ** max(-100, e - 1 if m == 0.5 else e)


def rotate(x, position, inv_freq, interleaved, scale):
    """x [..., D] of one token, float64; and the sum of magnitudes that each column is made of."""
    r = len(inv_freq)
    c, s = np.cos(position * inv_freq) * scale, np.sin(position * inv_freq) * scale
    ia, ib = (np.arange(0, 2 * r, 2), np.arange(1, 2 * r, 2)) if interleaved else (np.arange(r), np.arange(r, 2 * r))
    y, w = x.copy(), np.zeros_like(x)
    a, b = x[..., ia], x[..., ib]
    y[..., ia], y[..., ib] = a * c - b * s, b * c + a * s
    w[..., ia] = w[..., ib] = (np.abs(a) + np.abs(b)) * abs(scale)
    return y, w


def codes(x, scale):
    """Numbers over a scale, to the nearest e4m3 (what is no finite number becomes NaN), as float64."""
    y = torch.as_tensor(np.asarray(x, np.float64) / scale).float()
    y = torch.where(y.isfinite(), y, torch.nan)
    return y.to(E4M3).double().numpy()


def append(values, scales, x, slots, page):
    """values [P, H, page, D] codes as float64 and scales [P, H], updated; x [T, H, D] float64."""
    n_slots = values.shape[0] * page
    t = 0
    while t < len(slots):
        s = int(slots[t])
        if not 0 <= s < n_slots:
            t += 1
            continue
        p, at, n = s // page, s % page, 1
        while t + n < len(slots) and at + n < page and slots[t + n] == s + n:
            n += 1
        for h in range(values.shape[1]):
            rows = x[t:t + n, h]
            need = scale_for(np.abs(rows[np.isfinite(rows)]).max(initial=0.0))
            new = max(scales[p, h], need) if at else need
            if at and new != scales[p, h]:
                values[p, h, :at] = codes(values[p, h, :at] * scales[p, h], new)
            scales[p, h] = new
            values[p, h, at:at + n] = codes(rows, new)
        t += n


def attention(q, k, v, table, query_start, kv_len, page, scale, window, out_type):
    """q [T, Hq, D], k and v [P, H, page, D] float64 on the CPU (torch). Returns ({token: out [Hq, D]}, {token: bound [Hq, D]}): what of a
    kernel's roundings a result may have. Products are exact; a score's sum of D terms loses up to an ulp of its largest partial sum
    each term, 2^-23; weights are rounded to fp16, whose significand has 11 bits, so by up to 2^-11 of each (half a step, eps / 2),
    and made by an exponential of 2^-22; sums over n keys lose 2^-23 of what they hold in each of n / 16 steps and some joins."""
    heads, dim = q.shape[1], q.shape[2]
    kv_heads = k.shape[1]
    group = heads // kv_heads
    outs, bounds = {}, {}
    for i in range(len(kv_len)):
        first, last, n = int(query_start[i]), int(query_start[i + 1]), int(kv_len[i])
        last = min(last, q.shape[0])
        n = max(0, min(n, table.shape[1] * page))
        pages = [int(x) for x in table[i, :-(-n // page)]]
        there = np.repeat(np.array([0 <= x < k.shape[0] for x in pages], bool), page)[:n]
        safe = [x if 0 <= x < k.shape[0] else 0 for x in pages]
        keys = k[safe].permute(1, 0, 2, 3).reshape(kv_heads, -1, dim)[:, :n] if n else k.new_zeros(kv_heads, 0, dim)
        vals = v[safe].permute(1, 0, 2, 3).reshape(kv_heads, -1, dim)[:, :n] if n else v.new_zeros(kv_heads, 0, dim)
        at = np.arange(n)
        for t in range(first, last):
            pos = n - (last - first) + t - first
            see = there & (at <= pos) & ((at > pos - window) if window else True)
            see = torch.from_numpy(np.asarray(see, bool))
            if not see.any():
                outs[t], bounds[t] = torch.zeros(heads, dim, dtype=torch.float64), torch.zeros(heads, dim, dtype=torch.float64)
                continue
            kk, vv = keys[:, see], vals[:, see]
            x = q[t].view(kv_heads, group, dim)
            score = torch.einsum("hgd,hnd->hgn", x, kk) * scale
            size = (torch.einsum("hgd,hnd->hgn", x.abs(), kk.abs()) * abs(scale)).amax(2, keepdim=True)
            p = torch.softmax(score, 2)
            o = torch.einsum("hgn,hnd->hgd", p, vv)
            mass = torch.einsum("hgn,hnd->hgd", p, vv.abs())
            # weights lower than 2^-21 of the largest keep less: 2^-32 of the largest, at the largest scale
            tiny = 2.0 ** -30 * vv.abs().amax((1, 2)).view(kv_heads, 1, 1) * kk.shape[1] * p.amax(2, keepdim=True)
            e = half_ulp(out_type) * o.abs() + torch.finfo(out_type).tiny * torch.finfo(out_type).eps
            e = e + (2.0 ** -11 + 2 * size * dim * 2.0 ** -23 + 2.0 ** -19 + (kk.shape[1] / 16 + 64) * 2.0 ** -22) * mass + tiny
            outs[t], bounds[t] = o.reshape(heads, dim), (e * (1 + 2.0 ** -7)).reshape(heads, dim)
    return outs, bounds
