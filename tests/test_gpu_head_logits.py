"""The head with low-rank adapters beside it (mk_head_logits) against the 64-bit form. The bound is that of fp32 sums of exact
products, term by term (round_oracle.head)."""
import math

import numpy as np
import pytest
import torch

from tests import round_oracle as oracle

pytestmark = pytest.mark.gpu


def make(seed, rows, v, dim, rank, n, dtype, share=0.8):
    g = torch.Generator().manual_seed(seed)
    normal = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    c = {"hidden": normal(rows, dim).to(dtype), "weight": (normal(v, dim) / math.sqrt(dim)).to(dtype)}
    if n:
        c["down"] = (normal(n, rank, dim) / math.sqrt(dim)).to(dtype)
        c["up"] = (normal(n, v, rank) / math.sqrt(rank)).to(dtype)
        c["scale"] = torch.rand(n, generator=g) * 2
        c["adapter"] = torch.where(torch.rand(rows, generator=g) < share, torch.randint(0, n, (rows,), generator=g), -1).int()
    return c


def compare(sampler, c, hidden_pad=0, out_pad=0):
    f = lambda k: c[k].double().numpy() if k in c else None  # noqa: E731
    want, bound = oracle.head(f("hidden"), f("weight"), c["adapter"].numpy() if "adapter" in c else None, f("down"), f("up"), f("scale"))
    rows, dim = c["hidden"].shape
    v = c["weight"].shape[0]
    wide = torch.full((rows, dim + hidden_pad), math.nan, dtype=c["hidden"].dtype, device="cuda")
    hidden = wide[:, :dim]
    hidden.copy_(c["hidden"])
    room = torch.full((rows, v + out_pad), -77.0, device="cuda")
    rest = {k: c[k].cuda() for k in ("adapter", "down", "up", "scale") if k in c}
    got = sampler.head_logits(hidden, c["weight"].cuda(), out=room[:, :v], **rest)
    x = got.cpu().double().numpy()
    assert (room[:, v:] == -77.0).all()
    off = np.abs(x - want)
    assert (off <= bound).all(), (np.unravel_index((off - bound).argmax(), off.shape), off.max(), bound.max())
    return got


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows, v, dim, rank, n", [
    (1, 1, 8, 8, 1), (1, 4099, 64, 16, 1), (3, 127, 72, 8, 2), (16, 128, 128, 16, 3), (17, 1000, 200, 24, 5), (33, 515, 1032, 64, 4),
    (64, 2049, 512, 16, 16), (65, 300, 640, 128, 3), (100, 777, 64, 40, 7), (129, 1025, 320, 8, 40), (257, 400, 136, 32, 2),
    (300, 1300, 256, 16, 9), (512, 600, 192, 64, 5)])
def test_sizes(gpu_sampler_factory, dtype, rows, v, dim, rank, n):
    compare(gpu_sampler_factory(129280, 512), make(rows + v, rows, v, dim, rank, n, dtype))


def test_a_models_width(gpu_sampler_factory):
    """A long sum, and more columns than all CTAs take at once."""
    compare(gpu_sampler_factory(129280, 512), make(7, 24, 40000, 4096, 16, 6, torch.bfloat16))


@pytest.mark.parametrize("rows", [1, 40, 200])
def test_without_adapters(gpu_sampler_factory, rows):
    compare(gpu_sampler_factory(129280, 512), make(5, rows, 1000, 256, 0, 0, torch.bfloat16))
    c = make(6, rows, 1000, 256, 16, 3, torch.bfloat16, share=0.0)
    got = compare(gpu_sampler_factory(129280, 512), c)
    c["adapter"][:] = 3  # none of the three
    assert torch.equal(got, compare(gpu_sampler_factory(129280, 512), c))
    c["adapter"][:] = 0
    del c["scale"]
    compare(gpu_sampler_factory(129280, 512), c)


@pytest.mark.parametrize("hidden_pad, out_pad", [(8, 0), (64, 3), (0, 1), (24, 2)])
def test_strides(gpu_sampler_factory, hidden_pad, out_pad):
    """What lies behind a hidden state is NaN and has no part in it; what lies behind a row of logits stays."""
    compare(gpu_sampler_factory(129280, 512), make(9, 37, 1001, 200, 16, 3, torch.bfloat16), hidden_pad, out_pad)


def test_adapters_in_any_order(gpu_sampler_factory):
    """A row's logits are the same to the bit wherever it stands and whatever is beside it."""
    c = make(11, 96, 700, 256, 16, 6, torch.bfloat16, share=1.0)
    got = compare(gpu_sampler_factory(129280, 512), c)
    order = torch.randperm(96, generator=torch.Generator().manual_seed(1))
    d = dict(c, hidden=c["hidden"][order], adapter=c["adapter"][order])
    assert torch.equal(got[order.cuda()], compare(gpu_sampler_factory(129280, 512), d))


def test_a_rows_nan_stays_its_own(gpu_sampler_factory):
    c = make(13, 50, 900, 320, 16, 4, torch.float16, share=1.0)
    clean = compare(gpu_sampler_factory(129280, 512), c)
    c["hidden"][7] = math.nan
    c["hidden"][20, 3] = math.inf
    cuda = {k: x.cuda() for k, x in c.items()}
    got = gpu_sampler_factory(129280, 512).head_logits(**cuda)
    assert got[7].isnan().all() and not got[20].isfinite().any()
    other = [t for t in range(50) if t not in (7, 20)]
    assert torch.equal(got[other], clean[other])
    c = make(13, 50, 900, 320, 16, 4, torch.float16, share=0.5)
    c["up"][2, 100] = math.nan  # an adapter's, in one column
    got = gpu_sampler_factory(129280, 512).head_logits(**{k: x.cuda() for k, x in c.items()})
    bad = (c["adapter"] == 2).cuda()
    assert bad.any() and got[bad][:, 100].isnan().all() and not got[~bad].isnan().any() and not got[:, 101].isnan().any()


def test_streams_and_captures(gpu_sampler_factory):
    """Two graphs of one handle, of other sizes, replayed one behind the other on new inputs."""
    sampler = gpu_sampler_factory(129280, 512)
    graphs = []
    for rows, v in ((40, 1500), (7, 3333)):
        c = {k: x.cuda() for k, x in make(rows, rows, v, 384, 16, 4, torch.bfloat16).items()}
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        out = torch.empty(rows, v, device="cuda")
        with torch.cuda.stream(stream):
            sampler.head_logits(**c, out=out)
        stream.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            sampler.head_logits(**c, out=out)
        graphs.append((g, c, out))
    for g, c, out in graphs + graphs:
        c["hidden"].mul_(-0.5)
        c["adapter"].copy_(c["adapter"].flip(0))
        out.fill_(math.nan)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, sampler.head_logits(**c))


def test_refusals(gpu_sampler_factory):
    from mako_b200 import BatchSampler, MakoError
    sampler = BatchSampler(64, 4)
    z = lambda *n, t=torch.bfloat16: torch.zeros(*n, dtype=t, device="cuda")  # noqa: E731
    for h, w in ((z(5, 64), z(64, 64)), (z(4, 64), z(65, 64)), (z(4, 60), z(64, 60))):
        with pytest.raises(MakoError):
            sampler.head_logits(h, w)
    with pytest.raises(MakoError, match="16-byte"):
        sampler.head_logits(z(4, 72)[:, 4:68], z(64, 64))
    with pytest.raises(MakoError, match="multiples of 8"):
        sampler.head_logits(z(4, 68)[:, :64], z(64, 64))
    ids = z(4, t=torch.int32)
    for rank in (12, 136):
        with pytest.raises(MakoError, match="rank"):
            sampler.head_logits(z(4, 64), z(64, 64), adapter=ids, down=z(2, rank, 64), up=z(2, 64, rank))
    with pytest.raises(AssertionError):
        sampler.head_logits(z(4, 64), z(64, 64, t=torch.float16))
    with pytest.raises(AssertionError):
        sampler.head_logits(z(4, 64, t=torch.float32), z(64, 64, t=torch.float32))
    assert sampler.head_logits(z(0, 64), z(64, 64)).shape == (0, 64)
