"""The page plan (mk_kv_plan_step) at every number of sequences that it takes, whatever was called before or is called beside it."""
import subprocess
import sys
import threading

import numpy as np
import pytest
import torch

from tests import round_oracle as oracle
from tests import test_gpu_kv_plan as kv
from tests.conftest import ROOT

pytestmark = pytest.mark.gpu


def small(rng, s):
    return kv.make(rng, s, 16, 40, 3, 2 * s)


def run_sizes(sizes):
    from mako_b200 import BatchSampler
    sampler = BatchSampler(32, 1)
    rng = np.random.default_rng(1)
    for s in sizes:
        kv.both(lambda *_: sampler, *small(rng, s), 16, 2 * s)


def test_sizes_in_ascending_order():
    """In a process of its own: what a larger call has set before would help a smaller one."""
    sizes = [4029, 4030, 4031, 4032, 4095, 4096, 4097, 6000, 8191, 8192]
    code = f"from tests import test_gpu_plan_limits as t; t.run_sizes({sizes})"
    done = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=600)
    assert done.returncode == 0, done.stderr[-2000:]


def test_more_sequences_than_it_takes_are_refused(gpu_sampler_factory):
    from mako_b200 import MakoError
    with pytest.raises(MakoError, match="n_seq 8193"):
        kv.both(gpu_sampler_factory, *small(np.random.default_rng(2), 8193), 16, 9)


def test_two_threads_of_other_sizes():
    """A thread's plans do not take the room of another one's, each on a handle and a stream of its own."""
    from mako_b200 import BatchSampler
    errors = []

    def work(s, device_arrays, sampler, stream, start):
        try:
            with torch.cuda.stream(stream):
                start.wait()
                for _ in range(2500):
                    sampler.kv_plan(*device_arrays, page_size=16)
            stream.synchronize()
        except Exception as e:  # noqa: BLE001
            errors.append((s, e))

    threads, start = [], threading.Barrier(3)
    for s in (8192, 5000, 4200):
        z = lambda *n: torch.zeros(*n, dtype=torch.int32, device="cuda")  # noqa: E731
        arrays = (z(s, 4), z(s), z(8), z(1), z(s))
        threads.append(threading.Thread(target=work, args=(s, arrays, BatchSampler(32, 1), torch.cuda.Stream(), start)))
    torch.cuda.synchronize()
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors


def test_plans_of_one_handle_side_by_side(gpu_sampler_factory):
    """Four streams, one handle, arrays of their own: pages taken and given back, over and over."""
    from mako_b200 import KvPlan
    sampler, rng, work = gpu_sampler_factory(32, 1), np.random.default_rng(6), []
    for s in (300, 1000, 4500, 64):
        table, held, free, n_free, ln, nw = kv.make(rng, s, 16, 200, 9, 4 * s)
        held = -(-ln // 16)
        ids = rng.permutation(int(held.sum()) + 4 * s).astype(np.int32)
        table[:] = -1
        for i, at in enumerate(np.cumsum(held) - held):
            table[i, :held[i]] = ids[at:at + held[i]]
        free = np.concatenate([ids[held.sum():], np.full(held.sum(), -1, np.int32)])
        d = [torch.from_numpy(np.ascontiguousarray(x, dtype=np.int32)).cuda() for x in (table, held, free, [4 * s], ln)]
        want, _ = oracle.plan(table, held.astype(np.int32), free, 4 * s, ln, nw, 16, 9 * s)
        work.append((d, [x.clone() for x in d], torch.from_numpy(nw).cuda(), KvPlan.empty(s, 9 * s), want, torch.cuda.Stream()))
    torch.cuda.synchronize()
    for _ in range(40):
        for d, _, nw, plan, _, stream in work:
            with torch.cuda.stream(stream):
                sampler.kv_plan(*d, nw, page_size=16, out=plan)
                sampler.kv_plan(*d, page_size=16)
    torch.cuda.synchronize()
    for d, before, _, plan, want, _ in work:
        for x, y in zip(d, before):
            assert torch.equal(x, y)
        for k, x in want.items():
            assert np.array_equal(getattr(plan, k).cpu().numpy().astype(np.int64), np.asarray(x, dtype=np.int64)), k
