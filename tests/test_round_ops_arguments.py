"""What the serving round's Python entry points refuse of their tensors, on the CPU: tensors that say which device they are on, and a
handle that is none, so that a call whose tensors are taken ends at the library's own check."""
import pytest
import torch

from mako_b200 import BatchSampler, KvPlan, MakoError
from mako_b200 import sampler as module


class On(torch.Tensor):
    """A tensor that says it lies on device `where`."""
    where = 0

    def get_device(self):
        return self.where


def on(*size, t=torch.float32):
    return torch.zeros(*size, dtype=t).as_subclass(On)


@pytest.fixture
def handle(monkeypatch):
    h = BatchSampler.__new__(BatchSampler)
    h._h, h._index, h.device = None, 0, torch.device("cpu")
    monkeypatch.setattr(module, "_stream_ptr", lambda device: None)
    return h


def head(h):
    b = torch.bfloat16
    x = {"hidden": on(3, 64, t=b), "weight": on(9, 64, t=b), "adapter": on(3, t=torch.int32), "down": on(2, 8, 64, t=b),
         "up": on(2, 9, 8, t=b), "scale": on(2), "out": on(3, 9)}
    return x, lambda: h.head_logits(**x)


def verify(h):
    x = {"logits": on(6, 100), "drafts": on(2, 2, t=torch.int32), "u": on(2, 4), "temperature": on(2), "draft_logits": on(4, 100),
         "draft_temperature": on(2), "mask": on(6, 4, t=torch.int32)}
    return x, lambda: h.spec_verify(**x)


def plan(h):
    i = lambda *n: on(*n, t=torch.int32)  # noqa: E731
    x = {"block_table": i(2, 4), "n_pages": i(2), "free_list": i(8), "n_free": i(1), "cache_len": i(2), "n_new": i(2)}
    y = {"query_start": i(3), "kv_len": i(2), "positions": i(5), "slots": on(5, t=torch.int64), "token_seq": i(5), "flags": i(2)}
    z = {**x, **y}
    return z, lambda: h.kv_plan(**{k: z[k] for k in x}, page_size=16, out=KvPlan(**{k: z[k] for k in y}))


@pytest.mark.parametrize("call", [head, verify, plan])
def test_tensors_of_another_device_or_the_host_are_refused(handle, call):
    tensors, run = call(handle)
    with pytest.raises(MakoError, match="null argument"):
        run()
    for k, x in tensors.items():
        for where in (1, -1):
            x.where = where
            with pytest.raises(AssertionError):
                run()
                pytest.fail(k)
        x.where = 0


def test_a_mask_narrower_than_the_rows_is_refused(handle):
    tensors, run = verify(handle)
    run_with = lambda mask: (tensors.update(mask=mask), run())  # noqa: E731
    with pytest.raises(AssertionError, match="narrower"):
        run_with(on(6, 8, t=torch.int32)[:, :3])
    with pytest.raises(MakoError, match="null argument"):  # (else the library's own check)
        run_with(on(6, 8, t=torch.int32)[:, :4])
