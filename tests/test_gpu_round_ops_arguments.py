"""What the serving round's Python entry points take and refuse of their tensors."""
import numpy as np
import pytest
import torch

from tests import test_gpu_kv_plan as kv
from tests import test_gpu_spec_verify as verify

pytestmark = pytest.mark.gpu


def test_a_single_rows_stride_has_no_meaning(gpu_sampler_factory):
    """A row that is the transpose of a column has a row stride of 1."""
    sampler = gpu_sampler_factory(129280, 512)
    g = torch.Generator(device="cuda").manual_seed(1)
    row = lambda x: x.as_strided(x.shape, (1, 1))  # noqa: E731
    hidden = torch.randn(1, 64, device="cuda", generator=g).bfloat16()
    weight = torch.randn(50, 64, device="cuda", generator=g).bfloat16()
    want = sampler.head_logits(hidden, weight)
    out = torch.empty(1, 50, device="cuda")
    sampler.head_logits(row(hidden), weight, out=row(out))
    assert torch.equal(out, want)
    c = verify.case(3, 1, 0, 500, mask=0.5)
    x = [torch.as_tensor(c[k]).cuda() for k in ("logits", "drafts", "u", "temperature")]
    mask = torch.from_numpy(c["mask"].view(np.int32)).cuda()
    a, b = sampler.spec_verify(*x, mask=mask), sampler.spec_verify(row(x[0]), *x[1:], mask=row(mask))
    assert torch.equal(a.tokens, b.tokens) and torch.equal(a.logprob, b.logprob)
    c = verify.case(4, 1, 1, 500)
    x = [torch.as_tensor(c[k]).cuda() for k in ("logits", "drafts", "u", "temperature", "draft_logits")]
    a, b = sampler.spec_verify(*x[:4], draft_logits=x[4]), sampler.spec_verify(*x[:4], draft_logits=row(x[4]))
    assert torch.equal(a.tokens, b.tokens) and torch.equal(a.logprob, b.logprob)
    one = verify.case(5, 1, 0, 1)
    x = [torch.as_tensor(one[k]).cuda() for k in ("logits", "drafts", "u", "temperature")]
    assert sampler.spec_verify(x[0].as_strided((1, 1), (9, 9)), *x[1:]).next_token.tolist() == [0]
    i = lambda *n: torch.zeros(*n, dtype=torch.int32, device="cuda")  # noqa: E731
    table, free = i(1, 3) - 1, torch.arange(5, dtype=torch.int32, device="cuda")
    held, n_free = i(1), i(1) + 5
    plan = sampler.kv_plan(row(table), held, free, n_free, i(1) + 20, i(1) + 1, page_size=16, out=_plan(1, 4))
    assert table.tolist() == [[4, 3, -1]] and plan.slots.tolist() == [3 * 16 + 4, -1, -1, -1]


def _plan(s, t):
    from mako_b200 import KvPlan
    return KvPlan.empty(s, t)


def test_a_mask_narrower_than_the_rows_is_refused(gpu_sampler_factory):
    """Also where its row stride would be wide enough: what lies behind is not its own."""
    z = lambda *n, t=torch.float32: torch.zeros(*n, dtype=t, device="cuda")  # noqa: E731
    with pytest.raises(AssertionError):
        gpu_sampler_factory(129280, 512).spec_verify(z(4, 100), z(2, 1, t=torch.int32), z(2, 3), 1.0, mask=z(4, 8, t=torch.int32)[:, :3])
