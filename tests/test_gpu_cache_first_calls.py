"""The first call that a process makes of each operator around the cache, and of the log-probabilities, is a captured one."""
import subprocess
import sys

import pytest

from tests.conftest import ROOT

pytestmark = pytest.mark.gpu

CODE = """
import torch
from mako_b200 import BatchSampler, KvCache
h = BatchSampler(32, 1)
i = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")
cache, freq = KvCache.empty(20, 2, 16, 128), torch.rand(64, device="cuda")
qkv = torch.randn(80, 12, 128, device="cuda").bfloat16()
q, k, v = qkv.split([8, 2, 2], 1)
slots, positions = torch.arange(80, device="cuda"), torch.arange(80, dtype=torch.int32, device="cuda")
table, x, tokens = torch.arange(20, dtype=torch.int32, device="cuda").view(1, 20), torch.randn(9, 70000, device="cuda"), i(*range(9))
mask = i(*[-1] * (9 * 2188)).view(9, 2188)
def step():
    turned = h.kv_append(cache, k, v, slots, q=q, positions=positions, inv_freq=freq)
    return [turned, h.kv_attention(turned, cache, table, i0, n80), h.kv_attention(turned[:1], cache, table, i1, n80, max_new=1),
            h.token_logprobs(x, tokens, 0.7, top=5).logprob, h.token_logprobs(x.half(), tokens, top=20, mask=mask).top_logprobs]
i0, i1, n80 = i(0, 80), i(0, 1), i(80)
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    r = step()
g.replay()
torch.cuda.synchronize()
for a, b in zip([y.clone() for y in r], step()):
    assert torch.equal(a, b) and not a.isnan().any()
"""


def test_the_first_call_is_captured():
    done = subprocess.run([sys.executable, "-c", CODE], cwd=ROOT, capture_output=True, text=True, timeout=600)
    assert done.returncode == 0, done.stderr[-2000:]
