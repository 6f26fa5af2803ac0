"""The first call that a process makes of each operator of the serving round is a captured one."""
import subprocess
import sys

import pytest

from tests.conftest import ROOT

pytestmark = pytest.mark.gpu

CODE = """
import torch
from mako_b200 import BatchSampler, KvPlan
h = BatchSampler(9000, 8)
z = lambda *n, t=torch.int32: torch.zeros(*n, dtype=t, device="cuda")
hidden, weight = torch.randn(8, 64, device="cuda").bfloat16(), torch.randn(9000, 64, device="cuda").bfloat16()
down, up = torch.randn(2, 8, 64, device="cuda").bfloat16(), torch.randn(2, 9000, 8, device="cuda").bfloat16()
out, u = torch.empty(8, 9000, device="cuda"), torch.rand(4, 3, device="cuda")
s = 5000
pages, new, plan = (z(s, 4) - 1, z(s), torch.arange(s, dtype=torch.int32, device="cuda"), z(1) + s, z(s)), z(s) + 1, KvPlan.empty(s, s)
drafts, ids = z(4, 1), z(8)
def step():
    h.head_logits(hidden, weight, adapter=ids, down=down, up=up, out=out)
    r = h.spec_verify(out, drafts, u, 1.0)
    h.kv_plan(*pages, new, page_size=16, out=plan)
    return r
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    r = step()
g.replay()
torch.cuda.synchronize()
a = r.tokens.clone(), plan.slots.clone()
assert torch.equal(step().tokens, a[0]) and torch.equal(plan.slots, a[1]) and int(a[1].max()) >= 16 * (s - 1)
"""


def test_the_first_call_is_captured():
    done = subprocess.run([sys.executable, "-c", CODE], cwd=ROOT, capture_output=True, text=True, timeout=600)
    assert done.returncode == 0, done.stderr[-2000:]
