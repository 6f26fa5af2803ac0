"""The append behind tokens whose page has a scale of any kind, against 64 bits: codes and scales exactly."""
import numpy as np
import pytest
import torch

from tests import kv_oracle as oracle
from tests.test_gpu_kv_append import TYPES, cache_of, sampler  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("page,dim", [(16, 64), (40, 128)])
def test_scales_that_are_no_power_of_two(sampler, kind, page, dim):  # noqa: F811
    """Numbers on and around the borders between two codes, of a scale that stays and of one that gives way."""
    rng = np.random.default_rng(page)
    pages, heads = 24, 2
    cache = cache_of(rng, pages, heads, page, dim)
    scale = rng.uniform(0.002, 0.05, (pages, heads)).astype(np.float32)
    scale[::3] *= 1e-4  # these give way (below)
    scale[1::3] = 7 * 2.0 ** -8  # by which borders are numbers of either type: ties, which an inverse's rounding would break
    for s in (cache.k_scale, cache.v_scale):
        s.copy_(torch.from_numpy(scale))
    place, new = page // 2, 6
    slots = (np.arange(pages)[:, None] * page + place + np.arange(new)).reshape(-1)
    # a code's upper border times the scale, as near as the type comes, and its neighbours
    grid = torch.arange(0, 0x7e, dtype=torch.uint8).view(oracle.E4M3).double().numpy()
    border = (grid[1:] + grid[:-1]) / 2
    border = border[border < 220]  # 448 of the power of two below a scale: it stays
    x = border[rng.integers(0, len(border), (pages, new, 2 * heads, dim))] * np.tile(scale, 2).reshape(pages, 1, 2 * heads, 1) * rng.choice([-1.0, 1.0], (pages, new, 2 * heads, dim))
    x[::3] *= 1e4
    x = torch.from_numpy(x).to(TYPES[kind]).view(torch.int16)
    x = (x + torch.from_numpy(rng.integers(0, 2, x.shape).astype(np.int16))).view(TYPES[kind]).view(-1, 2 * heads, dim).cuda()
    want = [(y.double().cpu().numpy(), s.double().cpu().numpy()) for y, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale))]
    sampler.kv_append(cache, x[:, :heads], x[:, heads:], torch.from_numpy(slots).cuda())
    wide = x.double().cpu().numpy()
    for (codes, scales), part, y, s in zip(want, (wide[:, :heads], wide[:, heads:]), (cache.k, cache.v), (cache.k_scale, cache.v_scale)):
        oracle.append(codes, scales, part, slots, page)
        assert np.array_equal(s.double().cpu().numpy(), scales)
        assert np.array_equal(y.double().cpu().numpy(), codes)
