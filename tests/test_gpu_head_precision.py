"""How far the head's logits (mk_head_logits) are off at a model's width, where the bound of a sum term by term says little: the tensor
core's accumulator truncates, so a sum goes through it in runs of 512 terms, and the adapters' inner sums stay in fp32.

What a step of 16 products cuts, as test_what_a_step_cuts sees it: each product what lies below a quarter of an ulp of the largest of
them and the accumulator, then their sum what lies below an ulp; up to 16 / 4 + 1 = 5 ulps, of products of one sign and many bits 2.5 on
average."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DIM, V, RANK, N = 4096, 1500, 16, 3
ULP = 2.0 ** -23


def errors(sampler, hidden, weight, **adapters):
    got = sampler.head_logits(hidden, weight, **adapters).double()
    want = hidden.double() @ weight.double().t()
    for t, a in enumerate(adapters["adapter"].tolist() if adapters else []):
        if a >= 0:
            inner = adapters["down"][a].double() @ hidden[t].double()
            want[t] += float(adapters["scale"][a]) * (adapters["up"][a].double() @ inner)
    return (got - want).cpu().numpy(), want.cpu().numpy()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("at", [1, 16])
def test_what_a_step_cuts(gpu_sampler_factory, dtype, at):
    """1, and products of 2^-20 to 2^-29 beside it in the same step or in the next one."""
    for k in range(20, 30):
        x, w = torch.zeros(1, 64, device="cuda"), torch.zeros(16, 64, device="cuda")
        x[0, 0], w[:, 0] = 1.0, 1.0
        n = 15 if at == 1 else 16
        x[0, at:at + n], w[:, at:at + n] = 2.0 ** -(k // 2), 2.0 ** -(k - k // 2)
        got = gpu_sampler_factory(129280, 512).head_logits(x.to(dtype), w.to(dtype)).double()
        want = math.floor(n * 2.0 ** (23 - k)) if k <= 25 else 0
        assert (((got - 1.0) / ULP) == want).all(), (k, got)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows", [1, 40, 90, 150, 200, 330])
@pytest.mark.parametrize("adapters", [False, True])
def test_signs_in_any_order(gpu_sampler_factory, dtype, rows, adapters):
    """Products of variance 1 / 4096: 32 steps of 16 a run, after j of which the sum is about 0.8 sqrt(16 j / 4096); cut by an ulp each (a
    half as a rule, and the products' own cuts are of either sign) that makes 6 ulps of 1, over eight runs of either sign 17, 2.0e-6 of a
    logit. Through one accumulator 4.4e-6 was measured; with inner sums of 16 bits it is 1e-3."""
    g = torch.Generator(device="cuda").manual_seed(rows)
    normal = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    hidden, weight = normal(rows, DIM).to(dtype), (normal(V, DIM) / math.sqrt(DIM)).to(dtype)
    rest = {}
    if adapters:
        rest = {"adapter": torch.arange(rows, device="cuda", dtype=torch.int32) % N, "down": (normal(N, RANK, DIM) / math.sqrt(DIM)).to(dtype),
                "up": (normal(N, V, RANK) / math.sqrt(RANK)).to(dtype), "scale": torch.ones(N, device="cuda")}
    off, want = errors(gpu_sampler_factory(129280, 512), hidden, weight, **rest)
    assert math.sqrt(np.mean(off ** 2)) <= 17 * ULP * math.sqrt(np.mean(want ** 2))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows", [1, 40, 90, 150, 200, 330])
def test_all_of_one_sign(gpu_sampler_factory, dtype, rows):
    """Every cut goes the same way. After j of a run's 32 steps the sum is j / 32 of the run's: 5 x 16.5 ulps of it at most, on average
    (as an ulp is 2^-23 of the value or less) 2.5 x 16.5 at most, and eight roundings of half an ulp. Through one accumulator of 256
    steps it would be 2.5 x 128.5 times what an ulp is of the value; 66 ulps (bf16, whose products have few bits) and 195 were measured."""
    g = torch.Generator(device="cuda").manual_seed(rows)
    positive = lambda *s: torch.rand(*s, device="cuda", generator=g) + 0.5  # noqa: E731
    hidden, weight = positive(rows, DIM).to(dtype), (positive(V, DIM) / DIM).to(dtype)
    off, want = errors(gpu_sampler_factory(129280, 512), hidden, weight)
    assert np.abs(off / want).max() <= 86.5 * ULP
    assert abs(np.mean(off / want)) <= 45.25 * ULP
