"""What mk_token_logprobs writes: its outputs, all of them and nothing else. By the C entry, into the middle of larger buffers; each output may be left out."""
import ctypes as C

import numpy as np
import pytest
import torch

from tests import kv_oracle as oracle

pytestmark = pytest.mark.gpu
GUARD, MARK = 64, 0x5A5A5A5A


def guarded(n):
    x = torch.full((n + 2 * GUARD,), MARK, dtype=torch.int32, device="cuda")
    return x, x.data_ptr() + 4 * GUARD


def untouched(x, n):
    x = x.cpu()
    return (x[:GUARD] == MARK).all() and (x[GUARD + n:] == MARK).all()


@pytest.mark.parametrize("rows,vocab", [(1, 129280), (3, 4099), (7, 40000), (600, 1237)])
@pytest.mark.parametrize("given,top", [(0, 0), (1, 1), (1, 64), (3, 5), (33, 0), (300, 33)])
def test_nothing_beside_the_outputs(rows, vocab, given, top):
    from mako_b200 import BatchSampler, lib
    from mako_b200._lib import LogprobRowsC
    h = BatchSampler(32, 1)
    rng = np.random.default_rng(vocab + given + top)
    x = torch.from_numpy(rng.normal(0, 3, (rows, vocab)).astype(np.float32)).cuda().bfloat16()
    tokens = torch.from_numpy(rng.integers(-1, vocab, (rows, max(given, 1))).astype(np.int32)).cuda()[:, :given].contiguous()
    r = LogprobRowsC(x.data_ptr(), vocab, 1, rows, vocab, tokens.data_ptr() or None, given, top, None, 0.8, None, 0)
    sizes = [rows * given, rows, rows * top, rows * top, rows]
    want = None
    for left_out in (None, 0, 1, 2, 3, 4):
        outs = [guarded(n) for n in sizes]
        pointers = [None if i == left_out else p for i, (_, p) in enumerate(outs)]
        assert lib.mk_token_logprobs(h._h, C.byref(r), *pointers, None) == 0
        torch.cuda.synchronize()
        for i, ((buffer, _), n) in enumerate(zip(outs, sizes)):
            assert untouched(buffer, n), (left_out, i)
            inside = buffer[GUARD:GUARD + n]
            if i == left_out:
                assert (inside == MARK).all(), i
            elif want is not None:
                assert torch.equal(inside, want[i]), (left_out, i)
        if want is None:
            want = [buffer[GUARD:GUARD + n].clone() for (buffer, _), n in zip(outs, sizes)]
    assert (want[4] == 0).all()
    logits = x.double().cpu().numpy()
    for i in range(0, rows, 97):
        lp, entropy, ids, tops, bound, bound_h = oracle.logprobs(logits[i], tokens[i].tolist(), float(np.float32(0.8)), top)
        assert want[2].view(rows, top)[i].tolist() == ids.tolist()
        room = np.array([bound[t] if t >= 0 else 0.0 for t in tokens[i].tolist()])
        assert (np.abs(want[0].view(torch.float32).view(rows, given)[i].double().cpu().numpy() - lp) <= room).all()
        assert (np.abs(want[3].view(torch.float32).view(rows, top)[i].double().cpu().numpy() - tops) <= bound[ids]).all()
        assert abs(float(want[1].view(torch.float32)[i]) - entropy) <= bound_h
