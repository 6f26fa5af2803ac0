"""The operators of a serving round around the sampler, as measurable cases: the language model's head with the requests'
own low-rank adapters beside it, the verification of drafted tokens against the target's distribution, and the block tables
and slot maps of the next forward pass. One dict per case, inputs made on the GPU from a seed, the plain form by elementary
torch operations, and the same results in 64 bits.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # one request being decoded with its own adapter
        {"name": "head_1", "kind": "head", "rows": 1, "vocab": 129280, "dim": 4096, "rank": 16, "adapters": 1, "share": 1.0,
         "type": "bf16"},
        # a server's decode step: sixteen adapters among 64 requests, a quarter of which use none
        {"name": "head_64", "kind": "head", "rows": 64, "vocab": 129280, "dim": 4096, "rank": 16, "adapters": 16, "share": 0.75,
         "type": "bf16"},
        # a small model with a vocabulary and a width that fill no tile
        {"name": "head_odd", "kind": "head", "rows": 37, "vocab": 50257, "dim": 2056, "rank": 8, "adapters": 5, "share": 0.9,
         "type": "fp16"},
        # the rows of a speculative round, 64 sequences of five positions, with wide adapters
        {"name": "head_320", "kind": "head", "rows": 320, "vocab": 151552, "dim": 4096, "rank": 64, "adapters": 8, "share": 0.9,
         "type": "bf16"},
        # one sequence with four drafts
        {"name": "verify_1", "kind": "verify", "seqs": 1, "drafts": 4, "vocab": 129280, "type": "fp32", "temperature": 0.8,
         "noise": 1.0, "onehot": False, "mask": False, "ragged": False, "mixed": False},
        # a server's round, a drafter that samples
        {"name": "verify_64", "kind": "verify", "seqs": 64, "drafts": 4, "vocab": 129280, "type": "fp32", "temperature": 0.6,
         "noise": 1.0, "onehot": False, "mask": False, "ragged": False, "mixed": False},
        # drafts looked up in the context (no distribution behind them), grammar masks, requests with temperatures of their own
        {"name": "verify_lookup_128", "kind": "verify", "seqs": 128, "drafts": 3, "vocab": 151552, "type": "fp16",
         "temperature": 0.9, "noise": 0.5, "onehot": True, "mask": True, "ragged": True, "mixed": True},
        # many sequences with long drafts, 16-bit rows, the untruncated distribution
        {"name": "verify_256", "kind": "verify", "seqs": 256, "drafts": 7, "vocab": 151552, "type": "bf16", "temperature": 1.0,
         "noise": 0.5, "onehot": False, "mask": False, "ragged": True, "mixed": False},
        # a decode step: one token a sequence
        {"name": "pages_decode_256", "kind": "pages", "seqs": 256, "page": 16, "longest": 8192, "new": 1, "ragged": False},
        # a speculative round: up to eight tokens a sequence
        {"name": "pages_spec_1000", "kind": "pages", "seqs": 1000, "page": 32, "longest": 4096, "new": 8, "ragged": True},
        # prompts that are worked off in chunks
        {"name": "pages_prompts_48", "kind": "pages", "seqs": 48, "page": 64, "longest": 131072, "new": 2048, "ragged": True},
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["head", "verify", "pages"])
    if kind == "head":
        c = {"kind": kind, "rows": _log_int(rng, 1, 320), "vocab": _log_int(rng, 1000, 151552), "dim": 8 * _log_int(rng, 32, 896),
             "rank": rng.choice([8, 16, 24, 32, 64]), "adapters": _log_int(rng, 1, 24), "share": rng.choice([0.0, 0.5, 0.9, 1.0]),
             "type": rng.choice(["bf16", "fp16"])}
        while c["vocab"] * c["dim"] > 151552 * 4096:
            c["dim"] = 8 * _log_int(rng, 32, 512)
        return c
    if kind == "verify":
        c = {"kind": kind, "seqs": _log_int(rng, 1, 224), "drafts": rng.randint(0, 7), "vocab": _log_int(rng, 4000, 151552),
             "type": rng.choice(["fp32", "bf16", "fp16"]), "temperature": round(rng.uniform(0.3, 1.3), 2),
             "noise": round(rng.uniform(0.2, 1.2), 2), "onehot": rng.random() < 0.35, "mask": rng.random() < 0.4,
             "ragged": rng.random() < 0.6, "mixed": rng.random() < 0.4}
        while work(c)["bytes"] > 1.1e9:
            c["seqs"] = _log_int(rng, 1, 128)
        return c
    return {"kind": kind, "seqs": _log_int(rng, 1, 1000), "page": rng.choice([16, 24, 32, 64, 128]), "longest": _log_int(rng, 64, 65536),
            "new": _log_int(rng, 1, 64), "ragged": rng.random() < 0.7}


# ---- inputs --------------------------------------------------------------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed) * 7919 + 17)
    return g


def _prepare_head(c, g):
    t, rows, n = TYPES[c["type"]], c["rows"], c["adapters"]
    normal = lambda *s: torch.randn(*s, device=DEV, generator=g)  # noqa: E731
    weight = torch.empty(c["vocab"], c["dim"], dtype=t, device=DEV)
    weight.normal_(0.0, 2.0 / math.sqrt(c["dim"]), generator=g)
    hidden = normal(rows, c["dim"]).to(t)  # behind the last norm
    down = (normal(n, c["rank"], c["dim"]) / math.sqrt(c["dim"])).to(t)
    up = (normal(n, c["vocab"], c["rank"]) * (0.5 / math.sqrt(c["rank"]))).to(t)
    scale = 0.5 + 1.5 * torch.rand(n, device=DEV, generator=g)
    with_one = int(round(rows * c["share"]))
    order = torch.randperm(rows, device=DEV, generator=g)
    adapter = torch.full((rows,), -1, dtype=torch.int32, device=DEV)
    adapter[order[:with_one]] = torch.arange(with_one, device=DEV, dtype=torch.int32) % n
    return {"hidden": hidden, "weight": weight, "down": down, "up": up, "scale": scale, "adapter": adapter,
            "out": torch.empty(rows, c["vocab"], device=DEV)}


def _target_rows(n, v, g):
    """A head's output: N(0, 2^2) with eight spikes U(8, 15) a row."""
    x = torch.empty(n, v, device=DEV).normal_(0.0, 2.0, generator=g)
    at = torch.randint(0, v, (n, 8), device=DEV, generator=g)
    return x.scatter_(1, at, 8.0 + 7.0 * torch.rand(n, 8, device=DEV, generator=g))


def _pick(rows, temperature, g):
    """One token a row, drawn at the row's temperature."""
    noise = torch.empty_like(rows).exponential_(1.0, generator=g).log_()
    return (rows / temperature - noise).argmax(1)


def _prepare_verify(c, g):
    s, d, v, t = c["seqs"], c["drafts"], c["vocab"], TYPES[c["type"]]
    temperature = torch.full((s,), float(c["temperature"]), device=DEV)
    if c["mixed"]:  # requests' own temperatures, every fifth greedy
        temperature = 0.4 + 0.8 * torch.rand(s, device=DEV, generator=g)
        temperature[::5] = 0.0
    target = _target_rows(s * (d + 1), v, g).view(s, d + 1, v)
    near = (target[:, :d] + c["noise"] * torch.randn(s, d, v, device=DEV, generator=g)).reshape(s * d, v).to(t)
    each = temperature.clamp_min(1e-2).view(s, 1, 1).expand(s, d, 1).reshape(s * d, 1)
    mask, allowed = None, None
    if c["mask"]:  # a tenth of the vocabulary, two spikes of every row's among it
        words = (v + 31) // 32
        bits = torch.rand(s * (d + 1), words * 32, device=DEV, generator=g) < 0.1
        best = target.reshape(-1, v).topk(2, 1).indices
        bits.scatter_(1, best, True)
        bits[:, v:] = False
        weights = torch.tensor([1 << i for i in range(31)] + [-(1 << 31)], dtype=torch.int64, device=DEV)
        mask = (bits.view(s * (d + 1), words, 32).long() * weights).sum(2).to(torch.int32)
        allowed = bits[:, :v].reshape(s, d + 1, v)[:, :d].reshape(s * d, v)
    if d:
        seen = near.float()
        if allowed is not None:
            seen = seen.masked_fill(~allowed, -math.inf)
        drafts = _pick(seen, each, g).view(s, d).to(torch.int32)
    else:
        drafts = torch.empty(s, 0, dtype=torch.int32, device=DEV)
    if c["ragged"] and d:  # sequences whose drafter stopped early
        n = torch.randint(0, d + 1, (s, 1), device=DEV, generator=g)
        drafts.masked_fill_(torch.arange(d, device=DEV).view(1, d) >= n, -1)
    return {"logits": target.reshape(s * (d + 1), v).to(t), "draft_logits": None if c["onehot"] or not d else near,
            "drafts": drafts, "u": torch.rand(s, d + 2, device=DEV, generator=g), "temperature": temperature, "mask": mask}


def _prepare_pages(c, g):
    s, page = c["seqs"], c["page"]
    ints = lambda low, high: torch.randint(low, high, (s,), device=DEV, generator=g, dtype=torch.int32)  # noqa: E731
    cache_len = ints(1, c["longest"] + 1)
    n_new = ints(1, c["new"] + 1) if c["ragged"] else torch.full((s,), c["new"], dtype=torch.int32, device=DEV)
    if s > 8:  # requests that have ended, and ones that pause
        cache_len[3::16] = 0
        n_new[3::16] = 0
        n_new[5::16] = 0
    columns = -(-(c["longest"] + c["new"]) // page)
    held = ((cache_len + page - 1) // page).to(torch.int32)
    total = s * (columns + 1)
    ids = torch.randperm(total, device=DEV, generator=g).to(torch.int32)
    at = torch.arange(columns, device=DEV).view(1, columns)
    first = (held.long().cumsum(0) - held).view(s, 1)
    table = torch.where(at < held.view(s, 1), ids[(first + at).clamp_max(total - 1)], torch.full((), -1, dtype=torch.int32, device=DEV))
    used = held.sum(dtype=torch.int32)
    free = torch.arange(total, device=DEV)
    free = torch.where(free < total - used, ids[(free + used).clamp_max(total - 1)], -1)
    most = s * c["new"] + 5  # room for the fullest step, and a few rows of padding
    i32 = lambda n: torch.empty(n, dtype=torch.int32, device=DEV)  # noqa: E731
    return {"cache_len": cache_len, "n_new": n_new, "block_table": table.contiguous(), "n_pages": held, "free_list": free,
            "n_free": (total - used).view(1), "page": page, "max_tokens": most,
            "out": {"query_start": i32(s + 1), "kv_len": i32(s), "positions": i32(most),
                    "slots": torch.empty(most, dtype=torch.int64, device=DEV), "token_seq": i32(most), "flags": i32(s)}}


def prepare(case, seed):
    state = {"head": _prepare_head, "verify": _prepare_verify, "pages": _prepare_pages}[case["kind"]](case, _gen(seed))
    state["kind"] = case["kind"]
    return state


# ---- plain forms ---------------------------------------------------------------------------------------------------------------

def _plain_head(s):
    x, (n, rank, dim) = s["hidden"].float(), s["down"].shape
    inner = x @ s["down"].float().view(n * rank, dim).t()  # of every adapter, [rows][n * rank]
    of = torch.arange(n, device=DEV).repeat_interleave(rank)
    inner = inner * s["scale"][of] * (s["adapter"].view(-1, 1) == of)
    return x @ s["weight"].float().t() + inner @ s["up"].float().permute(0, 2, 1).reshape(n * rank, -1)


def _weights(rows, temperature):
    """Weights of the rows' tokens relative to each row's largest, and the largest; one token alone where greedy or infinite.
    In 64 bits: a token's place in the running sum of a whole vocabulary is next to others' everywhere."""
    x = rows.double()
    x = torch.where(x.isnan(), -math.inf, x)
    most, at = x.max(2, keepdim=True)
    w = ((x - most) / temperature).exp()
    one = (temperature <= 0) | (most == math.inf)
    w = torch.where(one, torch.zeros_like(w).scatter_(2, at, 1.0), w)
    return torch.where(most == -math.inf, 0.0, w)


def _plain_verify(s):
    n, d = s["drafts"].shape
    v = s["logits"].shape[1]
    rows, temperature = s["logits"].view(n, d + 1, v).double(), s["temperature"].double().view(n, 1, 1)
    allowed = torch.ones((), dtype=torch.bool, device=DEV).expand(n, d + 1, v)
    if s["mask"] is not None:
        words = s["mask"].view(n, d + 1, -1, 1)
        allowed = ((words >> torch.arange(32, device=DEV)) & 1).bool().view(n, d + 1, -1)[:, :, :v]
    p = _weights(rows.masked_fill(~allowed, -math.inf), temperature)
    mass = p.sum(2, keepdim=True)
    p = p / mass.clamp_min(1e-300)
    there = ((s["drafts"] >= 0) & (s["drafts"] < v)).long().cumprod(1).bool()
    token = s["drafts"].long().clamp(0, v - 1)
    if s["draft_logits"] is not None:
        q = _weights(s["draft_logits"].view(n, d, v).double().masked_fill(~allowed[:, :d], -math.inf), temperature)
        q = q / q.sum(2, keepdim=True).clamp_min(1e-300)
    else:
        q = torch.zeros(n, d, v, dtype=torch.float64, device=DEV).scatter_(2, token.unsqueeze(2), 1.0)
    u = s["u"].double()
    p_token, q_token = p[:, :d].gather(2, token.unsqueeze(2))[..., 0], q.gather(2, token.unsqueeze(2))[..., 0]
    kept = ((u[:, :d] * q_token < p_token) & there).long().cumprod(1).sum(1)
    refused = kept < there.long().sum(1)  # there was a draft at the position that ends the round
    who = torch.arange(n, device=DEV)
    last = p[who, kept]
    q = torch.cat([q, torch.zeros(n, 1, v, dtype=torch.float64, device=DEV)], 1)[who, kept] * refused.view(n, 1)
    rest = (last - q).clamp_min(0.0)
    rest = torch.where(rest.sum(1, keepdim=True) > 0, rest, last)
    run = rest.cumsum(1)
    want = u[who, kept + refused.long()].view(n, 1) * run[:, -1:]
    nth = torch.searchsorted(run, want, right=True)[:, 0]
    highest = v - 1 - (rest.flip(1) > 0).long().argmax(1)
    none = last.sum(1) <= 0
    next_token = torch.where(none, -1, torch.minimum(nth, highest))
    at = torch.arange(d + 1, device=DEV).view(1, d + 1)
    padded = torch.cat([token, torch.zeros(n, 1, dtype=torch.int64, device=DEV)], 1)
    tokens = torch.where(at < kept.view(n, 1), padded, torch.where(at == kept.view(n, 1), next_token.view(n, 1), -1))
    logprob = p.gather(2, tokens.clamp_min(0).unsqueeze(2))[..., 0].log().masked_fill(tokens < 0, 0.0)
    empty = ~allowed[who, kept].any(1)
    flags = none.int() * 0x4 + (none & empty).int() * 0x8
    return [kept.int(), next_token.int(), tokens.int(), logprob.float(), flags]


def _plain_plan(s, n_new, most):
    """A step's plan: (the outputs, and what it leaves of the pages)."""
    n, columns = s["block_table"].shape
    page, cap = s["page"], s["free_list"].numel()
    length, new, held, free = s["cache_len"].long(), n_new.long(), s["n_pages"].long(), s["n_free"].long()
    want = (length + new + page - 1) // page
    bad = (length < 0) | (new < 0) | (held < 0) | (held > columns) | (want > columns)
    over = ~bad & (new > 0) & (torch.where(bad, 0, new).cumsum(0) > most)
    part = ~bad & ~over
    give = torch.where(part, (held - want).clamp_min(0), 0)
    give = torch.where(free + give.sum() > cap, torch.zeros_like(give), give)
    given = give.sum()
    take = torch.where(part, (want - held).clamp_min(0), 0)
    lack = (take > 0) & (take.cumsum(0) > free + given)
    take = torch.where(lack, 0, take)
    new = torch.where(part & ~lack, new, 0)
    # pages given back go on top of the list, the first of them topmost; pages are taken from the top
    at = torch.arange(columns, device=DEV).view(1, columns)
    held2, keep = held.view(n, 1), (held - give).view(n, 1)
    back = (at >= keep) & (at < held2) & ~bad.view(n, 1)
    rank = (give.cumsum(0) - give).view(n, 1) + at - keep
    pages = s["free_list"].clone()
    top = free + given
    pages = torch.cat([pages, pages.new_zeros(1)])
    pages[torch.where(back, top - 1 - rank, cap).view(-1)] = s["block_table"].reshape(-1)
    pages = pages[:cap]
    fresh = (at >= held2) & (at < held2 + take.view(n, 1))
    rank = (take.cumsum(0) - take).view(n, 1) + at - held2
    table = torch.where(fresh, pages[(top - 1 - rank).clamp(0, cap - 1)], torch.where(back, -1, s["block_table"]))
    start = torch.cat([new.new_zeros(1), new.cumsum(0)])
    token = torch.arange(most, device=DEV)
    seq = torch.searchsorted(start[1:].contiguous(), token, right=True)
    real = token < start[-1]
    seq0 = seq.clamp_max(n - 1)
    position = length[seq0] + token - start[seq0]
    slot = table[seq0, (position // page).clamp(0, columns - 1)].long() * page + position % page
    i32 = torch.int32
    out = {"query_start": start.to(i32), "kv_len": torch.where(bad, 0, length + new).to(i32),
           "positions": torch.where(real, position, 0).to(i32), "slots": torch.where(real, slot, -1),
           "token_seq": torch.where(real, seq, -1).to(i32),
           "flags": bad.to(i32) * 0x200 + over.to(i32) * 0x400 + lack.to(i32) * 0x800}
    return out, {"block_table": table, "n_pages": (held - give + take).to(i32), "free_list": pages,
                 "n_free": (top - take.sum()).to(i32)}


def _plain_pages(s):
    out, after = _plain_plan(s, s["n_new"], s["max_tokens"])
    left = _plain_plan({**s, **after}, torch.zeros_like(s["n_new"]), 0)[1]
    return {**out, "left": left}


# ---- the framework's calls -----------------------------------------------------------------------------------------------------

_handles = {}


def _sampler(n_vocab, rows):
    """The handle that a user's program keeps."""
    from mako_b200 import BatchSampler
    key = (n_vocab, rows)
    if key not in _handles:
        _handles.clear()
        _handles[key] = BatchSampler(n_vocab, rows)
    return _handles[key]


def _own_head(s):
    sampler = _sampler(s["weight"].shape[0], s["hidden"].shape[0])
    return sampler.head_logits(s["hidden"], s["weight"], adapter=s["adapter"], down=s["down"], up=s["up"], scale=s["scale"],
                               out=s["out"])


def _own_verify(s):
    sampler = _sampler(s["logits"].shape[1], s["drafts"].shape[0])
    r = sampler.spec_verify(s["logits"], s["drafts"], s["u"], s["temperature"], draft_logits=s["draft_logits"], mask=s["mask"],
                            mask_drafts=True)
    return [r.n_kept, r.next_token, r.tokens, r.logprob, r.flags]


def _own_pages(s):
    from mako_b200 import KvPlan
    sampler = _sampler(32, 1)
    pages = (s["block_table"], s["n_pages"], s["free_list"], s["n_free"], s["cache_len"])
    plan = sampler.kv_plan(*pages, s["n_new"], page_size=s["page"], out=KvPlan(**s["out"]))
    sampler.kv_plan(*pages, page_size=s["page"])  # the round came to nothing: the pages go back
    return {"query_start": plan.query_start, "kv_len": plan.kv_len, "positions": plan.positions, "slots": plan.slots,
            "token_seq": plan.token_seq, "flags": plan.flags,
            "left": {"block_table": s["block_table"], "n_pages": s["n_pages"], "free_list": s["free_list"],
                     "n_free": s["n_free"]}}


def run(state):
    kind = state["kind"]
    if own:
        return {"head": _own_head, "verify": _own_verify, "pages": _own_pages}[kind](state)
    return {"head": _plain_head, "verify": _plain_verify, "pages": _plain_pages}[kind](state)


def work(case):
    c = case
    if c["kind"] == "head":
        with_one = int(round(c["rows"] * c["share"]))
        used = min(c["adapters"], with_one)
        small = c["rank"] * (c["vocab"] + c["dim"])
        return {"bytes": 2 * (c["vocab"] + c["rows"]) * c["dim"] + 2 * used * small + 4 * c["rows"] * (c["vocab"] + 1),
                "flops": 2 * c["rows"] * c["vocab"] * c["dim"] + 2 * with_one * small}
    if c["kind"] == "verify":  # every row once; a round that ends early needs fewer
        rows = c["seqs"] * (c["drafts"] + 1 + (0 if c["onehot"] else c["drafts"]))
        size = 4 if c["type"] == "fp32" else 2
        masks = c["seqs"] * (c["drafts"] + 1) * 4 * ((c["vocab"] + 31) // 32) if c["mask"] else 0
        return {"bytes": rows * c["vocab"] * size + masks + c["seqs"] * (16 * c["drafts"] + 32), "flops": 3 * rows * c["vocab"]}
    tokens = c["seqs"] * c["new"]
    columns = -(-(c["longest"] + c["new"]) // c["page"])
    return {"bytes": 16 * tokens + 40 * c["seqs"] + 8 * c["seqs"] * columns, "flops": 10 * tokens}


# ---- 64 bits -------------------------------------------------------------------------------------------------------------------

def _exact_head(c, s):
    out = s["hidden"].double() @ s["weight"].double().t()
    for a in range(c["adapters"]):
        rows = (s["adapter"] == a).nonzero()[:, 0]
        if rows.numel():
            inner = s["hidden"][rows].double() @ s["down"][a].double().t()
            out[rows] += float(s["scale"][a]) * (inner @ s["up"][a].double().t())
    return out


def _exact_verify(c, s):
    """Sequence by sequence and position by position, as a host would."""
    n, d, v = c["seqs"], c["drafts"], c["vocab"]

    def dist(row, t, allowed):
        x = row.double()
        if allowed is not None:
            x = torch.where(allowed, x, -math.inf)
        if t <= 0:
            return torch.nn.functional.one_hot(x.argmax(), v).double()
        return (x / t - torch.logsumexp(x / t, 0)).exp()

    token_of = s["drafts"].tolist()
    u, temperature = s["u"].double().tolist(), s["temperature"].double().tolist()
    kept, following, all_tokens, logs = [], [], [], []
    for i in range(n):
        chosen, lp, j, q = [], [], 0, None
        while True:
            allowed = None
            if s["mask"] is not None:
                words = s["mask"][i * (d + 1) + j].long() & 0xffffffff
                allowed = ((words.view(-1, 1) >> torch.arange(32, device=DEV)) & 1).bool().reshape(-1)[:v]
            p = dist(s["logits"][i * (d + 1) + j], temperature[i], allowed)
            q, draw_with = None, u[i][j]
            if j < d and token_of[i][j] >= 0:
                t = token_of[i][j]
                if s["draft_logits"] is None:
                    q = torch.zeros_like(p)
                    q[t] = 1.0
                else:
                    q = dist(s["draft_logits"][i * d + j], temperature[i], allowed)
                if u[i][j] * float(q[t]) < float(p[t]):
                    chosen.append(t)
                    lp.append(math.log(float(p[t])))
                    j += 1
                    continue
                draw_with = u[i][j + 1]
            rest = p if q is None else (p - q).clamp_min(0.0)
            if float(rest.sum()) <= 0:
                rest = p
            run = rest.cumsum(0)
            t = int((run <= draw_with * run[-1]).sum())
            t = min(t, int(rest.nonzero()[-1]))
            kept.append(j)
            following.append(t)
            all_tokens.append(chosen + [t] + [-1] * (d - j))
            logs.append(lp + [math.log(float(p[t]))] + [0.0] * (d - j))
            break
    i32 = lambda x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    return [i32(kept), i32(following), i32(all_tokens).view(n, d + 1), torch.tensor(logs, dtype=torch.float64).view(n, d + 1),
            torch.zeros(n, dtype=torch.int32)]


def exact(case, seed):
    if case["kind"] == "pages":  # whole numbers: the plain form is as exact as can be
        return None
    s = prepare(case, seed)
    return _exact_head(case, s) if case["kind"] == "head" else _exact_verify(case, s)
