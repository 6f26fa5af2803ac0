"""Plain 64-bit forms of the serving round's operators, written as a host would run them."""
from __future__ import annotations

import math

import numpy as np


def head(hidden, weight, adapter=None, down=None, up=None, scale=None):
    """(logits, bound on what fp32 sums of exact products may be off by): numpy float64 arrays in."""
    out = hidden @ weight.T
    size = np.abs(hidden) @ np.abs(weight).T
    if adapter is not None:
        for t, a in enumerate(adapter):
            if 0 <= a < len(down):
                f = 1.0 if scale is None else float(scale[a])
                out[t] += f * (up[a] @ (down[a] @ hidden[t]))
                size[t] += abs(f) * (np.abs(up[a]) @ (np.abs(down[a]) @ np.abs(hidden[t])))
    # a term passes through at most so many roundings of 2^-23 (a truncating sum's): the sum over dim, the inner sum over dim,
    # its scale and its sum over rank, and the two put together
    n = hidden.shape[1] + (0 if adapter is None else down.shape[2] + down.shape[1]) + 4
    return out, n * 2.0 ** -23 * size


def _dist(row, t, allowed):
    x = np.where(np.isnan(row), -math.inf, row.astype(np.float64))
    if allowed is not None:
        x = np.where(allowed, x, -math.inf)
    m = x.max()
    if m == -math.inf:
        return np.zeros_like(x)
    if not 0 < t < 1e30 or m == math.inf:
        w = np.zeros_like(x)
        w[int(x.argmax())] = 1.0
        return w
    with np.errstate(invalid="ignore"):
        w = np.where(x > -math.inf, np.exp((x - m) / t), 0.0)
    return w / w.sum()


def bits(words, n):
    return ((words.view(np.uint32)[:, None] >> np.arange(32, dtype=np.uint32)) & 1).astype(bool).reshape(-1)[:n]


def verify(logits, drafts, u, temperature, draft_logits=None, draft_temperature=None, mask=None, mask_drafts=False):
    """Per sequence: (n_kept, next_token, tokens, logprob, flags, margin): margin is how near any of its decisions came to the
    other side, as a part of the whole."""
    (n, d), v = drafts.shape, logits.shape[1]
    res = []
    for i in range(n):
        tp = float(temperature[i])
        tq = tp if draft_temperature is None else float(draft_temperature[i])
        chosen, logs, j, margin, flags = [], [], 0, 1.0, 0
        while True:
            row = i * (d + 1) + j
            allowed = None if mask is None else bits(mask[row], v)
            p = _dist(logits[row], tp, allowed)
            t = int(drafts[i, j]) if j < d else -1
            q, uu = np.zeros(v), float(u[i, j])
            if 0 <= t < v:
                if draft_logits is None:
                    q[t] = 1.0
                else:
                    q = _dist(draft_logits[i * d + j], tq, allowed if mask_drafts else None)
                margin = min(margin, abs(uu * q[t] - p[t]) or (0.0 if p[t] else 1.0))
                if uu * q[t] < p[t]:
                    chosen.append(t)
                    logs.append(math.log(p[t]))
                    j += 1
                    continue
                uu = float(u[i, j + 1])
            rest = np.maximum(p - q, 0.0)
            if rest.sum() <= 0:
                rest = p
            if rest.sum() <= 0:
                nxt, flags = -1, 0x4 | (0x8 if allowed is not None and not allowed.any() else 0)
            else:
                run = np.cumsum(rest)
                at = np.nonzero(run > uu * run[-1])[0]
                nxt = int(at[0]) if len(at) else int(np.nonzero(rest)[0][-1])
                margin = min(margin, float(np.min(np.abs(run[:-1] - uu * run[-1]), initial=1.0)) / run[-1] or 1.0)
            tokens = chosen + [nxt] + [-1] * (d - j)
            logs = logs + [math.log(p[nxt]) if nxt >= 0 else 0.0] + [0.0] * (d - j)
            res.append((j, nxt, tokens, logs, flags, margin))
            break
    return res


def plan(block_table, n_pages, free, n_free, cache_len, n_new, page, max_tokens):
    """One step, sequence by sequence, on copies. free: the whole array. Returns the outputs and what is left of the pages."""
    table, held, free = block_table.copy(), n_pages.copy(), free.copy()
    s, cols = table.shape
    n_free = min(max(int(n_free), 0), len(free))
    ln, new = [int(x) for x in cache_len], [int(x) for x in n_new]
    want = [-(-(a + b) // page) for a, b in zip(ln, new)]
    flags, seen = [0] * s, 0
    for i in range(s):
        if ln[i] < 0 or new[i] < 0 or held[i] < 0 or held[i] > cols or want[i] > cols or ln[i] + new[i] > 2 ** 31 - 1:
            flags[i] = 0x200
            continue
        seen += new[i]
        if new[i] > 0 and seen > max_tokens:
            flags[i] = 0x400
    give = [max(0, int(held[i]) - want[i]) if not flags[i] else 0 for i in range(s)]
    if n_free + sum(give) <= len(free):
        back = []
        for i in range(s):
            if give[i]:
                back += table[i, want[i]:held[i]].tolist()
                table[i, want[i]:held[i]] = -1
                held[i] = want[i]
        free[n_free:n_free + len(back)] = back[::-1]
        n_free += len(back)
    need = 0
    for i in range(s):
        if flags[i] or want[i] <= held[i]:
            continue
        need += want[i] - int(held[i])
        if need > n_free:
            flags[i] = 0x800
    top = n_free
    start, pos, slots, seqs, kv = [0], [], [], [], []
    for i in range(s):
        run = new[i] if not flags[i] else 0
        if not flags[i]:
            while held[i] < want[i]:
                top -= 1
                table[i, held[i]] = free[top]
                held[i] += 1
        for t in range(ln[i], ln[i] + run):
            pos.append(t)
            slots.append(int(table[i, t // page]) * page + t % page)
            seqs.append(i)
        start.append(start[-1] + run)
        kv.append(0 if flags[i] == 0x200 else ln[i] + run)
    pad = max_tokens - len(pos)
    return {"query_start": start, "kv_len": kv, "positions": pos + [0] * pad, "slots": slots + [-1] * pad,
            "token_seq": seqs + [-1] * pad, "flags": flags}, (table, held, free, top)
