"""Operators of a serving pass on either side of the forward pass, as measurable cases: the log-probabilities of given tokens
with the entropy and the likeliest alternatives, the append of rotated keys and values to a paged cache of 8 bits with a scale
for each page and head, and the attention over that cache. One dict per case, inputs made on the GPU from a seed, the plain form
by elementary torch operations, and the same results in 64 bits.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
CODES = torch.float8_e4m3fn
LARGEST = 448.0  # of the 8-bit values


def listed():
    return [
        # a request that asks for the alternatives of each token it is sent, one decode step
        {"name": "logprobs_1", "kind": "logprobs", "rows": 1, "vocab": 129280, "given": 1, "top": 5, "type": "fp32", "mask": False,
         "mixed": False},
        # a server's decode step under grammars, sampled at temperatures of the requests' own; labels whose probabilities are asked for
        {"name": "logprobs_odd", "kind": "logprobs", "rows": 137, "vocab": 50257, "given": 3, "top": 20, "type": "fp16", "mask": True,
         "mixed": True},
        # the scoring of prompts
        {"name": "logprobs_prompt", "kind": "logprobs", "rows": 2048, "vocab": 151552, "given": 1, "top": 5, "type": "bf16",
         "mask": False, "mixed": False},
        # a decode step's keys and values
        {"name": "append_decode", "kind": "append", "seqs": 64, "new": 1, "longest": 512, "q_heads": 32, "kv_heads": 8, "dim": 128,
         "rotary": 128, "interleaved": False, "page": 16, "type": "bf16", "ragged": False},
        # a speculative round's, a part of each head rotated, pages of an odd size
        {"name": "append_spec_odd", "kind": "append", "seqs": 100, "new": 8, "longest": 300, "q_heads": 28, "kv_heads": 4, "dim": 64,
         "rotary": 32, "interleaved": True, "page": 24, "type": "fp16", "ragged": True},
        # prompts that are worked off in chunks
        {"name": "append_prompts", "kind": "append", "seqs": 6, "new": 2048, "longest": 700, "q_heads": 32, "kv_heads": 8, "dim": 128,
         "rotary": 128, "interleaved": False, "page": 64, "type": "bf16", "ragged": True},
        # one request being decoded
        {"name": "attend_1", "kind": "attend", "seqs": 1, "new": 1, "longest": 2048, "even": True, "q_heads": 32, "kv_heads": 8, "dim": 128,
         "page": 16, "window": 0, "type": "bf16", "prompts": 0},
        # a server's decode step
        {"name": "attend_decode_64", "kind": "attend", "seqs": 64, "new": 1, "longest": 16384, "even": False, "q_heads": 32, "kv_heads": 8,
         "dim": 128, "page": 16, "window": 0, "type": "bf16", "prompts": 0},
        # two requests with long contexts
        {"name": "attend_long_2", "kind": "attend", "seqs": 2, "new": 1, "longest": 131072, "even": True, "q_heads": 64, "kv_heads": 8,
         "dim": 128, "page": 64, "window": 0, "type": "bf16", "prompts": 0},
        # a speculative round over a window, head groups and pages that fill no tile
        {"name": "attend_spec_odd", "kind": "attend", "seqs": 37, "new": 4, "longest": 6000, "even": False, "q_heads": 28, "kv_heads": 4,
         "dim": 64, "page": 24, "window": 2000, "type": "fp16", "prompts": 0},
        # a pass in which a few prompts' chunks go beside the others' decoding
        {"name": "attend_mixed", "kind": "attend", "seqs": 24, "new": 400, "longest": 4000, "even": False, "q_heads": 16, "kv_heads": 4,
         "dim": 128, "page": 32, "window": 0, "type": "bf16", "prompts": 3},
        # prompts that are worked off in chunks
        {"name": "attend_prompts", "kind": "attend", "seqs": 4, "new": 2048, "longest": 8192, "even": True, "q_heads": 32, "kv_heads": 8,
         "dim": 128, "page": 64, "window": 0, "type": "bf16", "prompts": 4},
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["logprobs", "append", "attend", "attend"])
    if kind == "logprobs":
        c = {"kind": kind, "rows": _log_int(rng, 1, 2048), "vocab": _log_int(rng, 1000, 151552), "given": rng.choice([1, 1, 2, 7]),
             "top": rng.choice([0, 1, 5, 20, 32]), "type": rng.choice(["fp32", "bf16", "fp16"]), "mask": rng.random() < 0.3,
             "mixed": rng.random() < 0.5}
        while work(c)["bytes"] > 6e8:
            c["rows"] = _log_int(rng, 1, 1500)
        return c
    group = rng.choice([1, 2, 4, 5, 7, 8])
    c = {"kind": kind, "seqs": _log_int(rng, 1, 200), "new": 1, "longest": 1, "q_heads": 0, "kv_heads": rng.choice([1, 2, 4, 8]),
         "dim": rng.choice([64, 128]), "page": rng.choice([16, 24, 32, 64, 128]), "type": rng.choice(["bf16", "fp16"])}
    c["q_heads"] = group * c["kv_heads"]
    if kind == "append":
        c |= {"new": rng.choice([1, 1, _log_int(rng, 2, 9), _log_int(rng, 10, 2000)]), "longest": _log_int(rng, 1, 400),
              "rotary": c["dim"] // rng.choice([1, 1, 2, 4]), "interleaved": rng.random() < 0.5, "ragged": rng.random() < 0.7}
        while c["seqs"] * (c["new"] + c["longest"]) * c["q_heads"] * c["dim"] > 5e7:
            c["seqs"], c["longest"] = max(1, c["seqs"] // 2), max(1, c["longest"] // 2)
        return c
    prompt = rng.random() < 0.4
    c |= {"new": _log_int(rng, 16, 2048) if prompt else rng.choice([1, 1, 1, 2, 4, 6]), "longest": _log_int(rng, 32, 100000),
          "even": rng.random() < 0.4, "window": rng.choice([0, 0, 0, 128, 1000]), "prompts": 0}
    if prompt:
        c["seqs"] = min(c["seqs"], 40)
        c["prompts"] = rng.randint(1, min(c["seqs"], 4))
    held = lambda: 2 * c["seqs"] * c["longest"] * c["kv_heads"] * c["dim"]  # noqa: E731
    while held() > 2.1e9 or work(c)["bytes"] > 1.1e9 or work(c)["flops"] > 3e11 or c["seqs"] * c["q_heads"] * c["new"] * c["longest"] > 2.1e9:
        c["longest"], c["seqs"] = max(32, c["longest"] * 2 // 3), max(1, c["seqs"] * 3 // 4, c["prompts"])
        c["new"] = min(c["new"], c["longest"]) if not prompt else max(16, c["new"] * 3 // 4)
    c["longest"] = max(c["longest"], c["new"])
    return c


# ---- inputs --------------------------------------------------------------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed) * 7919 + 29)
    return g


def _prepare_logprobs(c, g):
    """A head's output, N(0, 2^2) with eight spikes U(8, 15) a row; the tokens asked for are mostly among the likely ones."""
    n, v, t = c["rows"], c["vocab"], TYPES[c["type"]]
    x = torch.empty(n, v, device=DEV).normal_(0.0, 2.0, generator=g)
    at = torch.randint(0, v, (n, 8), device=DEV, generator=g)
    x.scatter_(1, at, 8.0 + 7.0 * torch.rand(n, 8, device=DEV, generator=g))
    tokens = torch.cat([at, torch.randint(0, v, (n, 8), device=DEV, generator=g)], 1)[:, 6:6 + c["given"]].to(torch.int32)
    if n > 20:  # places that are padded
        tokens[7::20, 0] = -1
    mask = None
    if c["mask"]:  # a fifth of the vocabulary, most of the spikes among it
        words = (v + 31) // 32
        bits = torch.rand(n, words * 32, device=DEV, generator=g) < 0.2
        bits.scatter_(1, at[:, 2:], True)
        bits[:, v:] = False
        weights = torch.tensor([1 << i for i in range(31)] + [-(1 << 31)], dtype=torch.int64, device=DEV)
        mask = (bits.view(n, words, 32).long() * weights).sum(2).to(torch.int32)
    temperature = 0.3 + 1.2 * torch.rand(n, device=DEV, generator=g) if c["mixed"] else torch.ones(n, device=DEV)
    return {"logits": x.to(t), "tokens": tokens.contiguous(), "temperature": temperature, "mask": mask, "top": c["top"]}


def _lengths(c, g):
    """(tokens in the cache before the pass, tokens of the pass) of each sequence."""
    s = c["seqs"]
    ints = lambda low, high: torch.randint(low, high, (s,), device=DEV, generator=g)  # noqa: E731
    if c["kind"] == "append":
        before = ints(0, c["longest"] + 1)
        new = ints(1, c["new"] + 1) if c["ragged"] else torch.full((s,), c["new"], device=DEV)
    else:
        new = torch.full((s,), c["new"], device=DEV)
        if c["prompts"]:
            new[c["prompts"]:] = 1
        elif c["new"] > 1 and not c["even"]:
            new = ints(1, c["new"] + 1)
        end = torch.full((s,), c["longest"], device=DEV) if c["even"] else ints(1, c["longest"] + 1)
        before = (end - new).clamp_min(0)
    if s > 20:  # requests that sit this pass out, and that have ended
        new[5::19] = 0
        before[9::19] = 0
        new[9::19] = 0
    return before, new


def _table(c, lengths, spare, g):
    """Pages of a pool in no order, -1 behind each sequence's."""
    s, page = c["seqs"], c["page"]
    held = (lengths + page - 1) // page
    columns = -(-(c["longest"] + c["new"]) // page)
    total = s * columns + spare
    ids = torch.randperm(total, device=DEV, generator=g).to(torch.int32)
    at = torch.arange(columns, device=DEV).view(1, columns)
    first = (held.cumsum(0) - held).view(s, 1)
    return torch.where(at < held.view(s, 1), ids[(first + at).clamp_max(total - 1)], -1).contiguous(), total


def _start(new):
    return torch.cat([new.new_zeros(1), new.cumsum(0)]).to(torch.int32)


def _cache(total, c, g):
    """(codes, scales) of a pool: values of about one, a page's largest of which its scale follows."""
    shape = (total, c["kv_heads"], c["page"], c["dim"])
    scale = torch.randint(-9, -6, shape[:2], device=DEV, generator=g).float().exp2()
    x = torch.empty(shape, dtype=torch.bfloat16, device=DEV).normal_(0.0, 90.0, generator=g)
    return x.clamp_(-LARGEST, LARGEST).to(CODES), scale


def _prepare_append(c, g):
    before, new = _lengths(c, g)
    table, total = _table(c, before + new, 1, g)
    s, page, t = c["seqs"], c["page"], TYPES[c["type"]]
    most = s * c["new"]  # a pass of so many rows, padded behind the last sequence
    start = _start(new).long()
    token = torch.arange(most, device=DEV)
    seq = torch.searchsorted(start[1:].contiguous(), token, right=True)
    real, seq = token < start[-1], seq.clamp_max(s - 1)
    position = torch.where(real, before[seq] + token - start[seq], 0)
    slots = torch.where(real, table[seq, position // page].long() * page + position % page, -1)
    position = torch.where(real, position + (100000 if c["new"] == 1 else 0), 0)  # long conversations, whose first pages are gone
    heads = c["q_heads"] + 2 * c["kv_heads"]
    qkv = torch.empty(most, heads, c["dim"], device=DEV).normal_(0.0, 1.0, generator=g)
    qkv *= torch.exp(0.5 * torch.randn(heads, c["dim"], device=DEV, generator=g))  # channels that are larger than others
    half = torch.arange(c["rotary"] // 2, device=DEV, dtype=torch.float64) * 2.0 / c["rotary"]
    k, k_scale = _cache(total, c, g)
    v, v_scale = _cache(total, c, g)
    return {"qkv": qkv.to(t), "q_heads": c["q_heads"], "kv_heads": c["kv_heads"], "positions": position.to(torch.int32), "slots": slots,
            "inv_freq": torch.pow(10000.0, -half).float(), "interleaved": c["interleaved"], "k": k, "v": v, "k_scale": k_scale,
            "v_scale": v_scale, "q_out": torch.zeros(most, c["q_heads"], c["dim"], dtype=t, device=DEV)}


def _prepare_attend(c, g):
    before, new = _lengths(c, g)
    table, total = _table(c, before + new, 1, g)
    k, k_scale = _cache(total, c, g)
    v, v_scale = _cache(total, c, g)
    most = c["new"] * c["seqs"] if not c["prompts"] else c["new"] * c["prompts"] + c["seqs"] - c["prompts"]
    q = torch.empty(most, c["q_heads"], c["dim"], device=DEV).normal_(0.0, 1.5, generator=g).to(TYPES[c["type"]])
    return {"q": q, "k": k, "v": v, "k_scale": k_scale, "v_scale": v_scale, "block_table": table, "query_start": _start(new),
            "kv_len": (before + new).to(torch.int32), "max_new": c["new"], "window": c["window"], "out": torch.zeros_like(q)}


def prepare(case, seed):
    state = {"logprobs": _prepare_logprobs, "append": _prepare_append, "attend": _prepare_attend}[case["kind"]](case, _gen(seed))
    state["kind"] = case["kind"]
    return state


# ---- plain forms ---------------------------------------------------------------------------------------------------------------

def _plain_logprobs(s):
    x, (n, v) = s["logits"].float(), s["logits"].shape
    allowed = x > -math.inf  # neither that nor NaN
    if s["mask"] is not None:
        words = s["mask"].view(n, -1, 1)
        allowed = allowed & ((words >> torch.arange(32, device=DEV, dtype=torch.int32)) & 1).bool().view(n, -1)[:, :v]
    x = torch.where(allowed, x, -math.inf)
    y = x / s["temperature"].view(n, 1)
    y = y - y.max(1, keepdim=True).values
    w = y.exp()
    mass = w.sum(1, keepdim=True)
    entropy = mass.log()[:, 0] - torch.where(w > 0, w * y, 0.0).sum(1) / mass[:, 0]
    logprob = y - mass.log()
    token = s["tokens"].long()
    given = logprob.gather(1, token.clamp(0, v - 1)).masked_fill((token < 0) | (token >= v), 0.0)
    # the largest, ties to the lowest id: a key that orders by both
    bits = (x + 0.0).view(torch.int32).long()
    key = torch.where(bits < 0, -(bits & 0x7fffffff), bits) * (1 << 20) + (v - 1 - torch.arange(v, device=DEV))
    ids = key.topk(s["top"], 1).indices if s["top"] else key[:, :0]
    top = logprob.gather(1, ids)
    return [given, entropy, torch.where(top > -math.inf, ids, -1).to(torch.int32), top]


def _values(codes, scale):
    """What codes stand for; a scale is a power of two, so that 16 bits hold them."""
    return codes.to(torch.bfloat16) * scale.to(torch.bfloat16).view(*scale.shape, 1, 1)


def _rotate(x, cos, sin, interleaved):
    """The first 2 * cos.shape[-1] columns of x [T, H, D] by angles [T, 1, rotary / 2]."""
    half = cos.shape[-1]
    a, b = (x[..., 0:2 * half:2], x[..., 1:2 * half:2]) if interleaved else (x[..., :half], x[..., half:2 * half])
    c, d = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack([c, d], -1).flatten(-2) if interleaved else torch.cat([c, d], -1)
    return torch.cat([turned, x[..., 2 * half:]], -1)


def _plain_store(x, slots, codes, scale):
    """x [T, H, D] into the pages of codes [P, H, page, D] with scales [P, H], in place."""
    pages, heads, size, dim = codes.shape
    real = slots >= 0
    page = torch.where(real, slots // size, pages)
    x = torch.where(real.view(-1, 1, 1), x, 0.0)
    largest = x.abs().amax(2)
    most = torch.zeros(pages + 1, heads, device=DEV).index_reduce_(0, page, largest, "amax")[:pages]
    first = torch.full((pages + 1,), size, dtype=torch.int64, device=DEV).index_reduce_(0, page, slots % size, "amin")[:pages]
    touched = torch.zeros(pages + 1, dtype=torch.bool, device=DEV).index_fill_(0, page, True)[:pages]
    mantissa, exponent = torch.frexp(most.double() / LARGEST)
    need = torch.ldexp(torch.ones_like(mantissa), (exponent - (mantissa == 0.5).int()).clamp_min(-100)).float()
    need = torch.where(most > 0, need, 2.0 ** -100)
    fresh = torch.where((touched & (first > 0)).view(-1, 1), torch.maximum(scale, need), need)
    new = torch.where(touched.view(-1, 1), fresh, scale)
    older = (touched.view(-1, 1, 1, 1)) & (torch.arange(size, device=DEV).view(1, 1, -1, 1) < first.view(-1, 1, 1, 1))
    ratio = torch.where(new > 0, scale / new, 1.0).view(pages, heads, 1, 1)
    codes.copy_(torch.where(older, codes.float() * ratio, codes.float()).to(CODES))
    scale.copy_(new)
    at = page.clamp_max(pages - 1)
    y = (x / new[at].unsqueeze(2)).to(CODES).view(torch.uint8)
    # rows that are padding write what the first token writes, once more
    flat = codes.view(torch.uint8).permute(0, 2, 1, 3)
    flat[torch.where(real, page, page[0]), torch.where(real, slots, slots[0]) % size] = torch.where(real.view(-1, 1, 1), y, y[:1])


def _plain_append(s):
    x, h, k = s["qkv"].float(), s["q_heads"], s["kv_heads"]
    angle = s["positions"].double().view(-1, 1, 1) * s["inv_freq"].double()
    cos, sin = angle.cos().float(), angle.sin().float()
    q = _rotate(x[:, :h], cos, sin, s["interleaved"])
    real = (s["slots"] >= 0).view(-1, 1, 1)
    q = torch.where(real, q, 0.0).to(s["qkv"].dtype)
    _plain_store(_rotate(x[:, h:h + k], cos, sin, s["interleaved"]), s["slots"], s["k"], s["k_scale"])
    _plain_store(x[:, h + k:], s["slots"], s["v"], s["v_scale"])
    return [q, _values(s["k"], s["k_scale"]), _values(s["v"], s["v_scale"]), s["k_scale"], s["v_scale"]]


def _plain_attend(s):
    (pages, h, size, d), (n, columns) = s["k"].shape, s["block_table"].shape
    total, heads, _ = s["q"].shape
    start, length, new = s["query_start"].long(), s["kv_len"].long(), s["max_new"]
    long, table = columns * size, s["block_table"].long().clamp_min(0)

    def rows(codes, scale):  # [n, h, long, d]
        x = codes.view(torch.uint8)[table].view(CODES).float() * scale[table].view(n, columns, h, 1, 1)
        return x.permute(0, 2, 1, 3, 4).reshape(n, h, long, d)

    number = start[1:] - start[:-1]
    at = torch.arange(new, device=DEV).view(1, new)
    row = (start[:-1].view(n, 1) + at).clamp_max(total - 1)
    q = s["q"][row].float().view(n, new, h, heads // h, d).permute(0, 2, 3, 1, 4).reshape(n, h, -1, d)
    score = q @ rows(s["k"], s["k_scale"]).transpose(2, 3) / math.sqrt(d)
    position = (length - number).view(n, 1) + at
    key = torch.arange(long, device=DEV).view(1, 1, long)
    seen = (key <= position.unsqueeze(2)) & (key < length.view(n, 1, 1)) & (at < number.view(n, 1)).unsqueeze(2)
    if s["window"]:
        seen = seen & (key > position.unsqueeze(2) - s["window"])
    score = score.view(n, h, heads // h, new, long).masked_fill(~seen.view(n, 1, 1, new, long), -math.inf)
    w = (score - score.amax(4, keepdim=True).clamp_min(-1e30)).exp()
    w = w / w.sum(4, keepdim=True).clamp_min(1e-30)
    values = torch.where((key < length.view(n, 1, 1)).view(n, 1, long, 1), rows(s["v"], s["v_scale"]), 0.0)
    y = (w.view(n, h, -1, long) @ values).view(n, h, heads // h, new, d).permute(0, 3, 1, 2, 4).reshape(n * new, heads, d)
    into = torch.where(at < number.view(n, 1), row, total).view(-1)
    out = torch.zeros(total + 1, heads, d, device=DEV)
    out[into] = y
    return out[:total].to(s["q"].dtype)


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


def _own_logprobs(s):
    sampler = _sampler(s["logits"].shape[1], 1)
    r = sampler.token_logprobs(s["logits"], s["tokens"], s["temperature"], top=s["top"], mask=s["mask"])
    return [r.logprob, r.entropy, r.top_ids, r.top_logprobs]


def _own_cache(s):
    from mako_b200 import KvCache
    return KvCache(s["k"], s["v"], s["k_scale"], s["v_scale"])


def _own_append(s):
    h, k = s["q_heads"], s["kv_heads"]
    q, keys, values = s["qkv"].split([h, k, k], 1)
    _sampler(32, 1).kv_append(_own_cache(s), keys, values, s["slots"], q=q, q_out=s["q_out"], positions=s["positions"],
                              inv_freq=s["inv_freq"], interleaved=s["interleaved"])
    return [s["q_out"], _values(s["k"], s["k_scale"]), _values(s["v"], s["v_scale"]), s["k_scale"], s["v_scale"]]


def _own_attend(s):
    return _sampler(32, 1).kv_attention(s["q"], _own_cache(s), s["block_table"], s["query_start"], s["kv_len"], max_new=s["max_new"],
                                        window=s["window"], out=s["out"])


def run(state):
    kind = state["kind"]
    if own:
        return {"logprobs": _own_logprobs, "append": _own_append, "attend": _own_attend}[kind](state)
    return {"logprobs": _plain_logprobs, "append": _plain_append, "attend": _plain_attend}[kind](state)


def _mean_lengths(c):
    """(cached tokens before the pass, tokens of the pass, pairs of a query and a key) of a mean case, all sequences together."""
    s = c["seqs"]
    if c["kind"] == "append":
        return s * c["longest"] / 2, s * (c["new"] + 1) / 2 if c["ragged"] else s * c["new"], 0
    end = c["longest"] if c["even"] else c["longest"] / 2
    if c["prompts"]:
        new, other = c["prompts"] * c["new"], s - c["prompts"]
    else:
        new, other = s * (c["new"] if c["even"] or c["new"] == 1 else (c["new"] + 1) / 2), 0
    seen = min(end, c["window"]) if c["window"] else end
    each = new / max(1, s - other)
    of_new = max(seen - each / 2, seen / 2) if not c["window"] else seen
    return s * min(end, seen + each), new + other, new * of_new + other * seen


def work(case):
    c = case
    if c["kind"] == "logprobs":
        size = 4 if c["type"] == "fp32" else 2
        mask = 4 * ((c["vocab"] + 31) // 32) if c["mask"] else 0
        return {"bytes": c["rows"] * (c["vocab"] * size + mask + 8 * c["given"] + 8 * c["top"] + 8), "flops": 5 * c["rows"] * c["vocab"]}
    cached, new, pairs = _mean_lengths(c)
    if c["kind"] == "append":  # a page of which a part is there already has its codes read and written where the scale grows
        return {"bytes": int(new * c["dim"] * (4 * c["q_heads"] + 2 * 3 * c["kv_heads"]) + 12 * new),
                "flops": int(new * c["dim"] * (3 * c["q_heads"] + 6 * c["kv_heads"]))}
    tokens = cached * (1 + 4 / c["page"] / c["dim"])
    return {"bytes": int(2 * tokens * c["kv_heads"] * c["dim"] + 4 * new * c["q_heads"] * c["dim"]),
            "flops": int(4 * pairs * c["q_heads"] * c["dim"])}


# ---- 64 bits -------------------------------------------------------------------------------------------------------------------

def _exact_logprobs(c, s):
    given, entropies, ids, tops = [], [], [], []
    order = torch.arange(c["vocab"], device=DEV)
    for i in range(c["rows"]):
        x = s["logits"][i].double()
        if s["mask"] is not None:
            words = s["mask"][i].long() & 0xffffffff
            x = torch.where(((words[order // 32] >> (order % 32)) & 1) == 1, x, -math.inf)
        lp = torch.log_softmax(x / s["temperature"][i].double(), 0)
        p = lp.exp()
        entropies.append(-(p * lp)[p > 0].sum() if c["mask"] else -torch.special.xlogy(p, p).sum())
        t = s["tokens"][i].long()
        given.append(torch.where(t >= 0, lp[t.clamp_min(0)], 0.0))
        if c["top"]:
            low = x.topk(c["top"]).values[-1]
            near = (x >= low).nonzero()[:, 0]  # by id, and stably by value
            best = near[x[near].sort(descending=True, stable=True).indices[:c["top"]]]
        else:
            best = order[:0]
        ids.append(best.to(torch.int32))
        tops.append(lp[best])
    return [torch.stack(given), torch.stack(entropies), torch.stack(ids), torch.stack(tops)]


def _power(e):
    """2^e of whole e from -127 to 127, exactly."""
    return torch.tensor([2.0 ** i for i in range(-127, 128)], dtype=torch.float64).to(DEV)[e.long() + 127]


def _nearest(x):
    """The 8-bit value (a sign, four bits of exponent, three of mantissa) nearest to x, ties to even; |x| is at most 448."""
    step = _power(torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -6))) - 3.0)
    return torch.round(x / step) * step


def _exact_append(c, s):
    x, h, kv = s["qkv"].double(), c["q_heads"], c["kv_heads"]
    angle = s["positions"].double().view(-1, 1, 1) * s["inv_freq"].double()
    turn = torch.polar(torch.ones_like(angle), angle)
    half = c["rotary"] // 2

    def rotated(y):
        pair = y[..., :2 * half].unflatten(-1, (half, 2) if c["interleaved"] else (2, half))
        z = torch.view_as_complex((pair if c["interleaved"] else pair.transpose(-1, -2)).contiguous()) * turn
        z = torch.view_as_real(z)
        return torch.cat([(z if c["interleaved"] else z.transpose(-1, -2)).flatten(-2), y[..., 2 * half:]], -1)

    slots = s["slots"].tolist()
    runs = []  # (page, first place, first token, tokens)
    for t, at in enumerate(slots):
        if at < 0:
            continue
        if runs and runs[-1][0] == at // c["page"] and t and slots[t - 1] == at - 1:
            runs[-1][3] += 1
        else:
            runs.append([at // c["page"], at % c["page"], t, 1])

    def stored(y, codes, scale):
        values, scale = codes.double() * scale.double().view(*scale.shape, 1, 1), scale.double()
        for page, place, t, n in runs:
            fresh = y[t:t + n].permute(1, 0, 2)
            most = fresh.abs().amax((1, 2))
            power = torch.round(torch.log2((most / LARGEST).clamp_min(2.0 ** -100)))  # that or the next one
            need = _power(power + (LARGEST * _power(power) < most))
            new = torch.maximum(scale[page], need) if place else need
            old = values[page, :, :place]
            at = new.view(-1, 1, 1)
            values[page, :, :place] = torch.where(at == scale[page].view(-1, 1, 1), old, _nearest(old / at) * at)
            values[page, :, place:place + n] = _nearest(fresh / at) * at
            values[page, :, place + n:] *= (at / scale[page].view(-1, 1, 1))  # behind the last token: codes of no meaning, left as they are
            scale[page] = new
        return values, scale

    q = torch.where((s["slots"] >= 0).view(-1, 1, 1), rotated(x[:, :h]), 0.0)
    (k, k_scale), (v, v_scale) = stored(rotated(x[:, h:h + kv]), s["k"], s["k_scale"]), stored(x[:, h + kv:], s["v"], s["v_scale"])
    return [q, k, v, k_scale, v_scale]


def _exact_attend(c, s):
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    start, length = s["query_start"].tolist(), s["kv_len"].tolist()
    group = c["q_heads"] // c["kv_heads"]
    for i in range(c["seqs"]):
        first, last, n = start[i], start[i + 1], length[i]
        if first == last:
            continue
        pages = s["block_table"][i, :-(-n // c["page"])].long()
        where = n - (last - first) + torch.arange(last - first, device=DEV).view(-1, 1)
        key = torch.arange(n, device=DEV).view(1, -1)
        hidden = key > where
        if c["window"]:
            hidden = hidden | (key <= where - c["window"])
        for j in range(c["kv_heads"]):
            k = (s["k"][pages, j].double() * s["k_scale"][pages, j].double().view(-1, 1, 1)).reshape(-1, c["dim"])[:n]
            v = (s["v"][pages, j].double() * s["v_scale"][pages, j].double().view(-1, 1, 1)).reshape(-1, c["dim"])[:n]
            q = s["q"][first:last, j * group:(j + 1) * group].double().transpose(0, 1)
            score = torch.matmul(q, k.t()) / c["dim"] ** 0.5
            p = torch.softmax(score.masked_fill(hidden, -math.inf), 2)
            out[first:last, j * group:(j + 1) * group] = torch.matmul(p, v).transpose(0, 1)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return {"logprobs": _exact_logprobs, "append": _exact_append, "attend": _exact_attend}[case["kind"]](case, s)
