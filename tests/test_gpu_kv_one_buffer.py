"""Queries, rotated queries and outputs beside one another in the rows of one buffer, which share no number."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_side_by_side():
    from mako_b200 import BatchSampler, KvCache
    sampler = BatchSampler(32, 1)
    heads, q_heads, dim, tokens = 2, 4, 64, 150
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    qkv = torch.randn(tokens, q_heads + 2 * heads, dim, device="cuda").bfloat16()
    slots, positions, freq = torch.arange(tokens, device="cuda"), torch.arange(tokens, dtype=torch.int32, device="cuda"), torch.rand(dim // 2, device="cuda")
    table, start, length = torch.arange(10, dtype=torch.int32, device="cuda").view(1, 10), i32(0, tokens), i32(tokens)
    kw = dict(positions=positions, inv_freq=freq)
    q, k, v = qkv.split([q_heads, heads, heads], 1)
    cache = KvCache.empty(10, heads, 16, dim)
    turned = sampler.kv_append(cache, k, v, slots, q=q, **kw)
    want = sampler.kv_attention(turned, cache, table, start, length, max_new=tokens)
    wide = torch.zeros(tokens + 2, 3 * q_heads + 2 * heads, dim, device="cuda").bfloat16()  # out | rotated | q | k | v
    rows = wide[1:-1]
    rows[:, 2 * q_heads:] = qkv
    out, rotated, q, k, v = rows.split([q_heads, q_heads, q_heads, heads, heads], 1)
    other = KvCache.empty(10, heads, 16, dim)
    sampler.kv_append(other, k, v, slots, q=q, q_out=rotated, **kw)
    sampler.kv_attention(rotated, other, table, start, length, max_new=tokens, out=out)
    assert torch.equal(rotated, turned) and torch.equal(out, want)
    assert torch.equal(rows[:, 2 * q_heads:], qkv) and (wide[0] == 0).all() and (wide[-1] == 0).all()
    for call in (lambda: sampler.kv_append(other, k, v, slots, q=q, q_out=rows[:, 2 * q_heads - 1:3 * q_heads - 1], **kw),
                 lambda: sampler.kv_attention(rotated, other, table, start, length, out=rows[:, 1:1 + q_heads])):
        with pytest.raises(RuntimeError, match="overlaps"):
            call()
