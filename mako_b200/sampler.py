"""Host-side mirror of the reference sampler's interface over the C ABI.

`SamplingParams` and `Sampler` carry the names, argument meaning and error behaviour of mako::gen::SamplingParams and
mako::gen::Sampler (src/gen/sampler.hpp:12-45): one row, own state, own generator. `BatchSampler` is the batched
form the GPU is built for: torch CUDA tensors in, torch CUDA tensors out, one kernel launch per call. Torch is used
for device memory and streams only.
"""
from __future__ import annotations

import ctypes as C
import math
from dataclasses import dataclass
from typing import Optional

import numpy as np
import torch

from . import _lib
from ._lib import (HeadC, KvCacheC, KvPagesC, KvPlanC, KvQueriesC, KvRowsC, LogprobRowsC, RotaryC, RowsC, SampleOutC, SpecRowsC, check,
                   lib)
from .params import SamplingParams


def check_sampling(p: SamplingParams) -> None:
    """The range checks the reference applies upstream (src/server/openai.cpp:316-328); raises ValueError."""
    c = p.to_c()
    if lib.mk_check_sampling(C.byref(c)) != 0:
        raise ValueError(lib.mk_last_error().decode())


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _stream_ptr(device: torch.device) -> int:
    return torch._C._cuda_getCurrentRawStream(device.index)


def _first(t: torch.Tensor, b: int) -> torch.Tensor:
    """The first b rows, as a tensor of its own for each call (of a whole one: 0.5 us, a slice takes 1.4)."""
    return t.detach() if t.shape[0] == b else t[:b]


def _row_stride(t: torch.Tensor) -> int:
    """From one row to the next, of rows whose columns lie side by side (a tensor of one row, or one column, may say any stride)."""
    (ld, unit), (n, columns) = t.stride(), t.shape
    assert unit == 1 or columns <= 1
    return ld if n > 1 else columns


class Sampler:
    """One row at a time, as the reference: Sampler(params, n_vocab, seed); sample(); verify(); accept()."""

    def __init__(self, params: SamplingParams, n_vocab: int, seed: int, device: int = 0):
        if n_vocab == 0:
            raise ValueError("sampler: empty vocabulary")  # std::invalid_argument in the reference
        self._h = C.c_void_p()
        c = params.to_c()
        check(lib.mk_row_sampler_create(C.byref(self._h), C.byref(c), n_vocab, seed, device))
        self.n_vocab = n_vocab
        self.params = params

    def __del__(self):
        h = getattr(self, "_h", None)
        if h:
            lib.mk_row_sampler_destroy(h)
            self._h = None

    def greedy(self) -> bool:
        return self.params.temperature <= 0.0

    def accept(self, token: int) -> None:
        check(lib.mk_row_sampler_accept(self._h, int(token)))

    @staticmethod
    def _row_ptr(logits, n_vocab: int):
        if isinstance(logits, torch.Tensor):
            assert logits.dtype == torch.float32 and logits.numel() >= n_vocab and logits.is_contiguous()
            return logits.data_ptr(), logits
        a = np.ascontiguousarray(logits, dtype=np.float32)
        assert a.size >= n_vocab
        return a.ctypes.data, a

    def sample(self, logits) -> int:
        p, keep = self._row_ptr(logits, self.n_vocab)
        tok = C.c_int32()
        check(lib.mk_row_sampler_sample(self._h, p, C.byref(tok)))
        del keep
        return tok.value

    def verify(self, logits, draft: int):
        """Returns (token, accepted) — the reference returns the token and sets `accepted` by reference."""
        p, keep = self._row_ptr(logits, self.n_vocab)
        tok, acc = C.c_int32(), C.c_int32()
        check(lib.mk_row_sampler_verify(self._h, p, int(draft), C.byref(acc), C.byref(tok)))
        del keep
        return tok.value, bool(acc.value)


@dataclass
class SampleResult:
    token: torch.Tensor
    prob: torch.Tensor
    flags: torch.Tensor
    n_cand: torch.Tensor
    cand_ids: Optional[torch.Tensor] = None
    cand_q: Optional[torch.Tensor] = None
    accepted: Optional[torch.Tensor] = None
    draft_token: Optional[torch.Tensor] = None


@dataclass
class SpecVerifyResult:
    n_kept: torch.Tensor
    next_token: torch.Tensor
    tokens: torch.Tensor
    logprob: torch.Tensor
    flags: torch.Tensor


@dataclass
class KvPlan:
    """What a forward pass over a paged cache is handed (mk_kv_plan): query_start [S + 1], kv_len [S], positions [T], token_seq
    [T], flags [S] int32 and slots [T] int64, T being the most tokens a pass may have."""
    query_start: torch.Tensor
    kv_len: torch.Tensor
    positions: torch.Tensor
    slots: torch.Tensor
    token_seq: torch.Tensor
    flags: torch.Tensor

    @classmethod
    def empty(cls, n_seq: int, max_tokens: int, device="cuda") -> "KvPlan":
        i32 = lambda n: torch.empty(n, dtype=torch.int32, device=device)  # noqa: E731
        return cls(i32(n_seq + 1), i32(n_seq), i32(max_tokens), torch.empty(max_tokens, dtype=torch.int64, device=device),
                   i32(max_tokens), i32(n_seq))


@dataclass
class TokenLogprobs:
    logprob: torch.Tensor
    entropy: torch.Tensor
    top_ids: torch.Tensor
    top_logprobs: torch.Tensor
    flags: torch.Tensor


@dataclass
class KvCache:
    """A paged cache of keys and values in 8 bits (mk_kv_cache): k and v [P, H, page, D] float8_e4m3fn or uint8 of one shape and
    one set of strides, columns side by side (a [P, page, H, D] tensor is taken as its transpose(1, 2)); k_scale and v_scale [P, H]
    float32. What stands in page p, head h is k[p, h] times k_scale[p, h]."""
    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor

    @classmethod
    def empty(cls, n_pages: int, n_heads: int, page_size: int, dim: int, device="cuda") -> "KvCache":
        codes = lambda: torch.zeros((n_pages, n_heads, page_size, dim), dtype=torch.float8_e4m3fn, device=device)  # noqa: E731
        scales = lambda: torch.zeros((n_pages, n_heads), dtype=torch.float32, device=device)  # noqa: E731
        return cls(codes(), codes(), scales(), scales())

    def _c(self, on: int) -> KvCacheC:
        k, v, ks, vs = self.k, self.v, self.k_scale, self.v_scale
        (pages, heads, page, dim), stride = k.shape, k.stride()
        assert k.get_device() == v.get_device() == ks.get_device() == vs.get_device() == on, f"a cache on {k.device}, the handle is on {on}"
        assert k.dtype == v.dtype and k.dtype in (torch.float8_e4m3fn, torch.uint8) and ks.dtype == vs.dtype == torch.float32
        assert v.shape == k.shape and v.stride() == stride and stride[3] == 1
        assert ks.shape == vs.shape == (pages, heads) and ks.is_contiguous() and vs.is_contiguous()
        # (of a single page, head or place a tensor may say any stride)
        token = stride[2] if page > 1 else dim
        return KvCacheC(k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(), stride[0] if pages > 1 else 0, stride[1] if heads > 1 else 0,
                        token, pages, heads, page, dim)


def _heads_ld(t: torch.Tensor) -> int:
    """From one token to the next, of a [T, H, D] tensor whose heads lie side by side."""
    n, heads, dim = t.shape
    ld, head, unit = t.stride()
    assert unit == 1 and (head == dim or heads == 1)
    return ld if n > 1 else heads * dim


_TYPE = {torch.float32: _lib.FP32, torch.bfloat16: _lib.BF16, torch.float16: _lib.FP16}


class BatchSampler:
    """Batched sampling on one GPU. All tensors live on `device`; outputs are allocated once and reused."""

    def __init__(self, n_vocab: int, max_batch: int, device: int = 0, cand_cap: int = 0):
        if n_vocab == 0:
            raise ValueError("sampler: empty vocabulary")
        self.device, self._index = torch.device("cuda", device), device
        self._h = C.c_void_p()
        check(lib.mk_sampler_create(C.byref(self._h), device, n_vocab, max_batch))
        self.n_vocab, self.max_batch, self.cand_cap = n_vocab, max_batch, cand_cap
        d = self.device
        self.token = torch.empty(max_batch, dtype=torch.int32, device=d)
        self.prob = torch.empty(max_batch, dtype=torch.float32, device=d)
        self.flags = torch.zeros(max_batch, dtype=torch.int32, device=d)
        self.n_cand = torch.zeros(max_batch, dtype=torch.int32, device=d)
        self.accepted = torch.zeros(max_batch, dtype=torch.int32, device=d)
        self.draft_token = torch.zeros(max_batch, dtype=torch.int32, device=d)
        self.cand_ids = torch.zeros((max_batch, cand_cap), dtype=torch.int32, device=d) if cand_cap else None
        self.cand_q = torch.zeros((max_batch, cand_cap), dtype=torch.float32, device=d) if cand_cap else None

    def __del__(self):
        h = getattr(self, "_h", None)
        if h:
            lib.mk_sampler_destroy(h)
            self._h = None

    def set_overlap(self, mode: int) -> None:
        """How the row kernel is launched behind the previous kernel of the stream (mk_sampler_set_overlap):
        0 plain stream order, 1 programmatic dependent launch, 2 the same with the per-row history tables built
        before the wait (the caller promises that the previous kernel writes no parameters, histories or biases)."""
        check(lib.mk_sampler_set_overlap(self._h, int(mode)))

    def set_split(self, on: bool) -> None:
        """Whether a call of at most 148 rows may have every row's columns split over up to 64 CTAs, the last of which draws
        (the default, where it is faster), or runs as one CTA per row (mk_sampler_set_split)."""
        check(lib.mk_sampler_set_split(self._h, 1 if on else 0))

    # -- argument marshalling -----------------------------------------------------------------------------------
    def _rows(self, logits: torch.Tensor, params, history=None, history_len=None, mask=None, bias=None,
              n_vocab=None, id_offset: int = 0) -> RowsC:
        assert logits.is_cuda and logits.dtype == torch.float32 and logits.dim() == 2
        (ld, unit), (batch, columns) = logits.stride(), logits.shape
        assert unit == 1
        r = RowsC()
        r.logits = logits.data_ptr()
        r.ld = ld
        r.batch = batch
        r.n_vocab = n_vocab if n_vocab is not None else columns
        r.id_offset = id_offset
        if history is not None:
            assert history.is_cuda and history.dtype == torch.int32 and history.dim() == 2 and history.stride(1) == 1
            r.history = history.data_ptr()
            r.history_ld = history.stride(0)
            r.n_history = history.shape[1]
            if history_len is not None:
                assert history_len.dtype == torch.int32 and history_len.is_cuda
                r.history_len = history_len.data_ptr()
        if mask is not None:
            assert mask.is_cuda and mask.dtype in (torch.int32, torch.uint32) and mask.dim() == 2
            r.mask = mask.data_ptr()
            r.mask_ld = mask.stride(0)
        if bias is not None:
            # bias: [batch, n_bias, 2] int32 view of (id, float bits) pairs
            assert bias.is_cuda and bias.dtype == torch.int32 and bias.dim() == 3 and bias.shape[2] == 2
            assert bias.is_contiguous()
            r.bias = bias.data_ptr()
            r.n_bias = bias.shape[1]
        if isinstance(params, torch.Tensor):
            assert params.is_cuda and params.dtype == torch.int32 and params.shape == (batch, 7)
            r.params_dev = params.data_ptr()
        else:  # field by field: a structure of its own to copy from takes three times as long
            p = r.params
            p.temperature, p.top_k, p.top_p, p.min_p = params.temperature, params.top_k, params.top_p, params.min_p
            p.presence_penalty, p.frequency_penalty = params.presence_penalty, params.frequency_penalty
            p.repetition_penalty = params.repetition_penalty
        return r

    def _here(self, *tensors: torch.Tensor) -> None:
        """Refuses what lies on the host or on another device than the handle: a kernel that follows such an address faults."""
        for t in tensors:
            assert t.get_device() == self._index, f"a tensor on device {t.device}, the handle is on {self.device}"

    def _out(self, batch: int) -> SampleOutC:
        o = SampleOutC()
        o.token = self.token.data_ptr()
        o.prob = self.prob.data_ptr()
        o.flags = self.flags.data_ptr()
        o.n_cand = self.n_cand.data_ptr()
        if self.cand_cap:
            o.cand_ids = self.cand_ids.data_ptr()
            o.cand_q = self.cand_q.data_ptr()
            o.cand_cap = self.cand_cap
        return o

    def _result(self, b: int, **kw) -> SampleResult:
        return SampleResult(_first(self.token, b), _first(self.prob, b), _first(self.flags, b), _first(self.n_cand, b),
                            _first(self.cand_ids, b) if self.cand_cap else None,
                            _first(self.cand_q, b) if self.cand_cap else None, **kw)

    # -- the operations -----------------------------------------------------------------------------------------
    def sample(self, logits, params, u=None, *, history=None, history_len=None, mask=None, bias=None) -> SampleResult:
        """Sampler::sample for every row (src/gen/sampler.cpp:75-84); u[b] is the row's uniform."""
        r = self._rows(logits, params, history, history_len, mask, bias)
        o = self._out(r.batch)
        check(lib.mk_sampler_sample_batch(self._h, C.byref(r), _ptr(u), C.byref(o), _stream_ptr(self.device)))
        return self._result(r.batch)

    def verify(self, logits, params, draft, u_accept, u_redraw, *, history=None, history_len=None, mask=None,
               bias=None) -> SampleResult:
        """Sampler::verify for every row (src/gen/sampler.cpp:86-107)."""
        r = self._rows(logits, params, history, history_len, mask, bias)
        o = self._out(r.batch)
        check(lib.mk_sampler_verify_batch(self._h, C.byref(r), _ptr(draft), _ptr(u_accept), _ptr(u_redraw),
                                          C.byref(o), self.accepted.data_ptr(), _stream_ptr(self.device)))
        return self._result(r.batch, accepted=self.accepted[: r.batch])

    def verify_pq(self, target_logits, draft_logits, params, u_draft, u_accept, u_resample, *, history=None,
                  history_len=None, mask=None, bias=None) -> SampleResult:
        """Rejection sampling of a drafter's token against max(0, p - q)."""
        r = self._rows(target_logits, params, history, history_len, mask, bias)
        assert draft_logits.is_cuda and draft_logits.dtype == torch.float32 and draft_logits.stride(1) == 1
        b = r.batch
        check(lib.mk_sampler_verify_pq_batch(self._h, C.byref(r), draft_logits.data_ptr(), draft_logits.stride(0),
                                             _ptr(u_draft), _ptr(u_accept), _ptr(u_resample),
                                             self.draft_token.data_ptr(), self.accepted.data_ptr(),
                                             self.token.data_ptr(), self.flags.data_ptr(),
                                             _stream_ptr(self.device)))
        return SampleResult(self.token[:b], self.prob[:b], self.flags[:b], self.n_cand[:b],
                            accepted=self.accepted[:b], draft_token=self.draft_token[:b])

    def draft_pick(self, logits, head, embed, x, w, prev):
        """One step of the drafter pick (src/kernels/dsv41.metal:664-742) for up to 8 sequences: logits [S, V],
        head [V, rank], embed [E, rank], x [S, dim], w [dim + rank], prev [S] int32. Returns (draft [S] int32,
        conf [S] float32)."""
        for t in (logits, head, embed, x, w):
            assert t.is_cuda and t.dtype == torch.float32 and t.stride(-1) == 1
        assert head.is_contiguous() and embed.is_contiguous() and w.is_contiguous()
        n_seq, v = logits.shape
        rank, dim = head.shape[1], x.shape[1]
        assert head.shape[0] == v and embed.shape[1] == rank and w.numel() == dim + rank
        draft = torch.empty(n_seq, dtype=torch.int32, device=self.device)
        conf = torch.empty(n_seq, dtype=torch.float32, device=self.device)
        check(lib.mk_draft_pick(self._h, logits.data_ptr(), logits.stride(0), head.data_ptr(), embed.data_ptr(),
                                x.data_ptr(), x.stride(0), w.data_ptr(), prev.data_ptr(), n_seq, v, rank, dim,
                                embed.shape[0], draft.data_ptr(), conf.data_ptr(), _stream_ptr(self.device)))
        return draft, conf

    def draft_pick_plain(self, logits, h, conf_w, conf_bias: float, next_prev=None):
        """hy4_draft_pick (src/kernels/hy4f.metal:352-397): (argmax of each row with the lowest index on ties,
        sigmoid(conf_w . h[b] + conf_bias)). logits [S, V], h [S, width], conf_w [width]."""
        for t in (logits, h, conf_w):
            assert t.is_cuda and t.dtype == torch.float32 and t.stride(-1) == 1
        n_seq, v = logits.shape
        draft = torch.empty(n_seq, dtype=torch.int32, device=self.device)
        conf = torch.empty(n_seq, dtype=torch.float32, device=self.device)
        check(lib.mk_draft_pick_plain(self._h, logits.data_ptr(), logits.stride(0), n_seq, v, h.data_ptr(), h.stride(0),
                                      conf_w.data_ptr(), conf_w.numel(), float(conf_bias), draft.data_ptr(),
                                      conf.data_ptr(), _ptr(next_prev), _stream_ptr(self.device)))
        return draft, conf

    def rank_force(self, logits: torch.Tensor, token: torch.Tensor, k: int = 3):
        """ReasoningBudget::forced's logit test (src/server/openai.cpp:596-603) for every row: returns (forced [B]
        int32: token[b] if fewer than k raw logits are greater than its own, else -1; above [B]: that count)."""
        assert logits.is_cuda and logits.dtype == torch.float32 and logits.stride(1) == 1
        b, v = logits.shape
        forced = torch.empty(b, dtype=torch.int32, device=self.device)
        above = torch.empty(b, dtype=torch.int32, device=self.device)
        check(lib.mk_rank_force(self._h, logits.data_ptr(), logits.stride(0), b, v, token.data_ptr(), k,
                                forced.data_ptr(), above.data_ptr(), _stream_ptr(self.device)))
        return forced, above

    def decode_commit(self, sampled: torch.Tensor, history: torch.Tensor, history_len: torch.Tensor, *, forced=None,
                      next_input=None, flags=None) -> torch.Tensor:
        """One decode step's bookkeeping on the device (src/gen/session.cpp:416-444): forced tokens replace sampled
        ones, the token is appended to each row's history (history [B, cap] int32, history_len [B] int32, both
        updated in place) and written to next_input. Returns the committed tokens [B]."""
        b = sampled.shape[0]
        assert history.dtype == torch.int32 and history_len.dtype == torch.int32 and history.stride(1) == 1
        committed = torch.empty(b, dtype=torch.int32, device=self.device)
        check(lib.mk_decode_commit(self._h, b, sampled.data_ptr(), _ptr(forced), history.data_ptr(), history.stride(0),
                                   history.shape[1], history_len.data_ptr(), _ptr(next_input), committed.data_ptr(),
                                   _ptr(flags), _stream_ptr(self.device)))
        return committed

    def spec_resolve(self, accepted: torch.Tensor, token: torch.Tensor):
        """accepted/token: [n_seq, n_pos] int32. Returns (n_kept [n_seq], next_token [n_seq])."""
        n_seq, n_pos = accepted.shape
        kept = torch.empty(n_seq, dtype=torch.int32, device=self.device)
        nxt = torch.empty(n_seq, dtype=torch.int32, device=self.device)
        check(lib.mk_spec_resolve(self._h, n_seq, n_pos, accepted.data_ptr(), token.data_ptr(), kept.data_ptr(),
                                  nxt.data_ptr(), _stream_ptr(self.device)))
        return kept, nxt

    def spec_round(self, logits, params, drafts, u, *, history=None, history_len=None, forced=None, mask=None,
                   bias=None):
        """One speculative round of the reference (src/gen/session.cpp:451-506) for every sequence in one launch.
        logits [n_seq * n_pos, V]: row s*n_pos + j follows the round's token and drafts 0..j-1; drafts [n_seq,
        n_pos - 1] int32; u [n_seq, n_pos + 1] the sequence's uniforms in generator order; history [n_seq, cap] and
        history_len [n_seq] per sequence; forced [n_seq, n_pos] int32 (token or -1) or None. Returns (n_kept [n_seq],
        next_token [n_seq], result with per-position token / accepted / flags)."""
        n_seq, n_drafts = drafts.shape
        n_pos = n_drafts + 1
        assert logits.shape[0] == n_seq * n_pos and drafts.dtype == torch.int32 and drafts.is_contiguous()
        assert u.shape == (n_seq, n_pos + 1) and u.dtype == torch.float32 and u.is_contiguous()
        if forced is not None:
            assert forced.shape == (n_seq, n_pos) and forced.dtype == torch.int32 and forced.is_contiguous()
        r = self._rows(logits, params, history, history_len, mask, bias)
        o = self._out(r.batch)
        kept = torch.empty(n_seq, dtype=torch.int32, device=self.device)
        nxt = torch.empty(n_seq, dtype=torch.int32, device=self.device)
        check(lib.mk_sampler_spec_round(self._h, C.byref(r), n_pos, drafts.data_ptr(), _ptr(forced), u.data_ptr(),
                                        C.byref(o), self.accepted.data_ptr(), kept.data_ptr(), nxt.data_ptr(),
                                        _stream_ptr(self.device)))
        return kept, nxt, self._result(r.batch, accepted=self.accepted[: r.batch])

    def spec_commit(self, drafts, n_kept, next_token, history, history_len, *, next_input=None, flags=None) -> None:
        """The round's bookkeeping on the device: kept drafts, then next_token, appended to each sequence's history
        (history [n_seq, cap] and history_len [n_seq] updated in place); next_input receives next_token."""
        n_seq, n_drafts = drafts.shape
        check(lib.mk_spec_commit(self._h, n_seq, n_drafts + 1, drafts.data_ptr(), n_kept.data_ptr(),
                                 next_token.data_ptr(), history.data_ptr(), history.stride(0), history.shape[1],
                                 history_len.data_ptr(), _ptr(next_input), _ptr(flags), _stream_ptr(self.device)))

    # -- the round around the sampler -----------------------------------------------------------------------------
    def head_logits(self, hidden, weight, *, adapter=None, down=None, up=None, scale=None, out=None) -> torch.Tensor:
        """The model's head with the requests' low-rank adapters beside it (mk_head_logits): hidden [T, D], weight [V, D],
        down [N, R, D], up [N, V, R] bf16 or fp16, adapter [T] int32 (-1: none), scale [N] float32. Returns the rows that the
        sampler reads, [T, V] float32 (`out` where given)."""
        (rows, dim), v = hidden.shape, weight.shape[0]
        self._here(hidden, weight)
        assert hidden.dtype in (torch.bfloat16, torch.float16)
        assert weight.dtype == hidden.dtype and weight.is_contiguous() and weight.shape[1] == dim
        d_ptr = u_ptr = s_ptr = n = rank = 0
        if adapter is not None:
            self._here(adapter, down, up)
            assert adapter.dtype == torch.int32 and adapter.is_contiguous() and adapter.numel() == rows
            n, rank, _ = down.shape
            assert down.dtype == up.dtype == hidden.dtype
            assert down.shape == (n, rank, dim) and up.shape == (n, v, rank) and down.is_contiguous() and up.is_contiguous()
            d_ptr, u_ptr = down.data_ptr(), up.data_ptr()
            if scale is not None:
                self._here(scale)
                assert scale.dtype == torch.float32 and scale.is_contiguous() and scale.numel() == n
                s_ptr = scale.data_ptr()
        h = HeadC(weight.data_ptr(), d_ptr or None, u_ptr or None, s_ptr or None, v, dim, n, rank, _TYPE[hidden.dtype])
        if out is None:
            out = torch.empty((rows, v), dtype=torch.float32, device=hidden.device)
        self._here(out)
        assert out.dtype == torch.float32 and out.shape == (rows, v)
        check(lib.mk_head_logits(self._h, C.byref(h), hidden.data_ptr(), _row_stride(hidden), _ptr(adapter), rows, out.data_ptr(),
                                 _row_stride(out), _stream_ptr(self.device)))
        return out

    def spec_verify(self, logits, drafts, u, temperature, *, draft_logits=None, draft_temperature=None, mask=None,
                    mask_drafts: bool = False) -> SpecVerifyResult:
        """A speculative round against whole distributions (mk_spec_verify): logits [S * n_pos, V], drafts [S, n_pos - 1] int32
        (negative: no more drafts), u [S, n_pos + 1], temperature a number or [S] float32, draft_logits [S * (n_pos - 1), V] of
        the target's type or None for drafts that are certain, mask [S * n_pos, words]. Returns n_kept [S], next_token [S],
        tokens [S, n_pos], logprob [S, n_pos], flags [S]."""
        n_seq, n_drafts = drafts.shape
        n_pos, v = n_drafts + 1, logits.shape[1]
        self._here(logits, drafts, u)
        assert logits.shape[0] == n_seq * n_pos
        assert drafts.dtype == torch.int32 and drafts.is_contiguous()
        assert u.shape == (n_seq, n_pos + 1) and u.dtype == torch.float32 and u.is_contiguous()
        q_ptr = q_ld = t_ptr = t_all = qt_ptr = m_ptr = m_ld = 0
        if draft_logits is not None:
            self._here(draft_logits)
            assert draft_logits.dtype == logits.dtype and draft_logits.shape == (n_seq * n_drafts, v)
            q_ptr, q_ld = draft_logits.data_ptr(), _row_stride(draft_logits)
        if isinstance(temperature, torch.Tensor):
            self._here(temperature)
            assert temperature.dtype == torch.float32 and temperature.shape == (n_seq,) and temperature.is_contiguous()
            t_ptr = temperature.data_ptr()
        else:
            t_all = temperature
        if draft_temperature is not None:
            self._here(draft_temperature)
            assert draft_temperature.dtype == torch.float32
            assert draft_temperature.shape == (n_seq,) and draft_temperature.is_contiguous()
            qt_ptr = draft_temperature.data_ptr()
        if mask is not None:
            self._here(mask)
            assert mask.dtype in (torch.int32, torch.uint32) and mask.shape[0] == n_seq * n_pos
            m_ptr, m_ld = mask.data_ptr(), _row_stride(mask)
            assert 32 * mask.shape[1] >= v or m_ld == mask.shape[1], "a mask narrower than its rows"  # (the library sees strides alone)
        r = SpecRowsC(logits.data_ptr(), _row_stride(logits), q_ptr or None, q_ld, _TYPE[logits.dtype], n_seq, n_pos, v,
                      drafts.data_ptr(), u.data_ptr(), t_ptr or None, qt_ptr or None, t_all, m_ptr or None, m_ld, int(mask_drafts))
        kept, nxt, flags = torch.empty((3, n_seq), dtype=torch.int32, device=self.device).unbind()
        tokens = torch.empty((n_seq, n_pos), dtype=torch.int32, device=self.device)
        logprob = torch.empty((n_seq, n_pos), dtype=torch.float32, device=self.device)
        check(lib.mk_spec_verify(self._h, C.byref(r), kept.data_ptr(), nxt.data_ptr(), tokens.data_ptr(), logprob.data_ptr(),
                                 flags.data_ptr(), _stream_ptr(self.device)))
        return SpecVerifyResult(kept, nxt, tokens, logprob, flags)

    def kv_plan(self, block_table, n_pages, free_list, n_free, cache_len, n_new=None, *, page_size: int,
                out: Optional[KvPlan] = None) -> Optional[KvPlan]:
        """Pages, positions and slots of the next forward pass from the sequences' lengths, on the device (mk_kv_plan_step):
        block_table [S, columns], n_pages [S], free_list [P] and n_free [1] int32 are updated in place; cache_len [S] tokens are
        in the cache, n_new [S] come with the pass (None: pages above the need go back, and that is all). Fills and returns
        `out` (KvPlan.empty)."""
        (n_seq, cols), ld, i32 = block_table.shape, _row_stride(block_table), torch.int32
        assert block_table.dtype == n_pages.dtype == free_list.dtype == n_free.dtype == cache_len.dtype == i32
        on = self._index  # (as _here does, in one expression: a plan's time is its host's)
        assert block_table.get_device() == n_pages.get_device() == free_list.get_device() == n_free.get_device() == on
        assert cache_len.get_device() == on
        assert n_pages.is_contiguous() and cache_len.is_contiguous() and free_list.is_contiguous()
        assert n_pages.numel() == cache_len.numel() == n_seq and n_free.numel() == 1
        p = KvPagesC(block_table.data_ptr(), ld, cols, n_pages.data_ptr(), free_list.data_ptr(), free_list.numel(),
                     n_free.data_ptr(), page_size)
        if n_new is not None:
            assert n_new.get_device() == on and n_new.dtype == i32 and n_new.is_contiguous() and n_new.numel() == n_seq
            assert out is not None
        if out is None:
            o = KvPlanC()
        else:
            start, kv_len, pos, slots, seq, flags = out.query_start, out.kv_len, out.positions, out.slots, out.token_seq, out.flags
            assert start.get_device() == kv_len.get_device() == pos.get_device() == slots.get_device() == on
            assert seq.get_device() == flags.get_device() == on
            t = pos.numel()
            assert start.numel() == n_seq + 1 and kv_len.numel() == flags.numel() == n_seq and slots.numel() == seq.numel() == t
            assert start.dtype == kv_len.dtype == pos.dtype == seq.dtype == flags.dtype == i32 and slots.dtype == torch.int64
            assert start.is_contiguous() and kv_len.is_contiguous() and pos.is_contiguous() and slots.is_contiguous()
            assert seq.is_contiguous() and flags.is_contiguous()
            o = KvPlanC(start.data_ptr(), kv_len.data_ptr(), pos.data_ptr(), slots.data_ptr(), seq.data_ptr(), flags.data_ptr(), t)
        check(lib.mk_kv_plan_step(self._h, C.byref(p), cache_len.data_ptr(), _ptr(n_new), n_seq, C.byref(o),
                                  _stream_ptr(self.device)))
        return out

    def token_logprobs(self, logits, tokens, temperature=1.0, *, top: int = 0, mask=None) -> TokenLogprobs:
        """Log-probabilities of given tokens (mk_token_logprobs): logits [T, V] float32, bf16 or fp16, tokens [T] or [T, N] int32 (a
        negative one: none, 0), temperature a number or [T] float32, mask [T, words]. Returns logprob, of tokens' shape, entropy
        [T], the `top` likeliest tokens of each row, the likeliest first, in top_ids [T, top] with top_logprobs [T, top], and flags [T]."""
        rows, v = logits.shape
        self._here(logits, tokens)
        assert tokens.dtype == torch.int32 and tokens.is_contiguous() and tokens.dim() in (1, 2) and tokens.shape[0] == rows
        given = tokens.shape[1] if tokens.dim() == 2 else 1
        t_ptr = t_all = m_ptr = m_ld = 0
        if isinstance(temperature, torch.Tensor):
            self._here(temperature)
            assert temperature.dtype == torch.float32 and temperature.shape == (rows,) and temperature.is_contiguous()
            t_ptr = temperature.data_ptr()
        else:
            t_all = temperature
        if mask is not None:
            self._here(mask)
            assert mask.dtype in (torch.int32, torch.uint32) and mask.shape[0] == rows
            m_ptr, m_ld = mask.data_ptr(), _row_stride(mask)
            assert 32 * mask.shape[1] >= v, "a mask narrower than its rows"
        r = LogprobRowsC(logits.data_ptr(), _row_stride(logits), _TYPE[logits.dtype], rows, v, tokens.data_ptr(), given, top, t_ptr or None,
                         t_all, m_ptr or None, m_ld)
        f32, like = torch.float32, tokens.new_empty  # (0.5 us less each than torch.empty with a device)
        out = TokenLogprobs(like(tokens.shape, dtype=f32), like(rows, dtype=f32), like((rows, top)), like((rows, top), dtype=f32), like(rows))
        check(lib.mk_token_logprobs(self._h, C.byref(r), out.logprob.data_ptr(), out.entropy.data_ptr(), out.top_ids.data_ptr(),
                                    out.top_logprobs.data_ptr(), out.flags.data_ptr(), _stream_ptr(self.device)))
        return out

    def kv_append(self, cache: KvCache, k, v, slots, *, q=None, q_out=None, positions=None, inv_freq=None, interleaved: bool = False,
                  rotary_scale: float = 1.0):
        """A pass's keys and values into the cache (mk_kv_append): k and v [T, H, D] bf16 or fp16 at slots [T] int64 (negative:
        padding, left out), as kv_plan gives them. With inv_freq [R / 2] float32 the first R columns of k and of q [T, Hq, D] turn by
        positions [T] int32 times inv_freq, columns i and i + R / 2 or, interleaved, 2i and 2i + 1, and are scaled by rotary_scale.
        Returns q_out (rotated queries; q itself may be given), or None without q. k, v and q may be slices of one projection."""
        tokens, heads, dim = k.shape
        self._here(k, v, slots)
        assert k.dtype in (torch.bfloat16, torch.float16) and v.dtype == k.dtype and v.shape == k.shape
        assert slots.dtype == torch.int64 and slots.shape == (tokens,) and slots.is_contiguous()
        c = cache._c(self._index)
        assert (heads, dim) == (c.n_heads, c.dim)
        r = KvRowsC(k.data_ptr(), v.data_ptr(), _heads_ld(k), _heads_ld(v), None, None, 0, 0, 0, _TYPE[k.dtype], tokens, None, slots.data_ptr())
        if q is not None:
            q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device) if q_out is None else q_out
            self._here(q, q_out)
            assert q.dtype == q_out.dtype == k.dtype and q.shape == q_out.shape and q.shape[0] == tokens and q.shape[2] == dim
            r.q, r.q_out, r.q_ld, r.q_out_ld, r.n_q_heads = q.data_ptr(), q_out.data_ptr(), _heads_ld(q), _heads_ld(q_out), q.shape[1]
        else:
            assert q_out is None
        turn = None
        if inv_freq is not None:
            self._here(inv_freq, positions)
            assert inv_freq.dtype == torch.float32 and inv_freq.is_contiguous() and inv_freq.dim() == 1
            assert positions.dtype == torch.int32 and positions.shape == (tokens,) and positions.is_contiguous()
            r.positions = positions.data_ptr()
            turn = C.byref(RotaryC(inv_freq.data_ptr(), 2 * inv_freq.numel(), int(interleaved), rotary_scale))
        check(lib.mk_kv_append(self._h, C.byref(c), C.byref(r), turn, _stream_ptr(self.device)))
        return q_out

    def kv_attention(self, q, cache: KvCache, block_table, query_start, kv_len, *, max_new: int = 0, scale=None, window: int = 0,
                     out=None) -> torch.Tensor:
        """A pass's queries over the cache (mk_kv_attention): q [T, Hq, D] bf16 or fp16, block_table [S, columns], query_start
        [S + 1] and kv_len [S] int32 as kv_plan gives them; max_new: the most tokens that a sequence has in this pass, where the
        caller knows (it chooses kernels, nothing else); scale of a score, 1 / sqrt(D) by default; window: how many keys a token sees,
        its own among them (0: all). Returns [T, Hq, D] (`out` where given, apart from q); rows that are no sequence's are left as they are."""
        (tokens, q_heads, dim), (n_seq, cols) = q.shape, block_table.shape
        if out is None:
            out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        self._here(q, out, block_table, query_start, kv_len)
        assert q.dtype in (torch.bfloat16, torch.float16) and out.dtype == q.dtype and out.shape == q.shape
        assert block_table.dtype == query_start.dtype == kv_len.dtype == torch.int32
        assert query_start.is_contiguous() and kv_len.is_contiguous() and query_start.numel() == n_seq + 1 and kv_len.numel() == n_seq
        c = cache._c(self._index)
        assert c.dim == dim
        r = KvQueriesC(q.data_ptr(), out.data_ptr(), _heads_ld(q), _heads_ld(out), q_heads, _TYPE[q.dtype], tokens, block_table.data_ptr(),
                       _row_stride(block_table), cols, query_start.data_ptr(), kv_len.data_ptr(), n_seq, max_new,
                       1.0 / math.sqrt(dim) if scale is None else scale, window)
        r.workspace_bytes = lib.mk_kv_attention_bytes(C.byref(c), C.byref(r))
        # (of the caching allocator: a call's own, on its stream, and in a capture the graph's)
        workspace = torch.empty(r.workspace_bytes, dtype=torch.uint8, device=self.device)
        r.workspace = workspace.data_ptr()
        check(lib.mk_kv_attention(self._h, C.byref(c), C.byref(r), _stream_ptr(self.device)))
        return out

    def vp_local(self, shard_logits, params, k: int, records: torch.Tensor, *, id_offset: int, history=None,
                 history_len=None, mask=None, bias=None) -> torch.Tensor:
        """Vocab-parallel step 1: this shard's per-row record (max, sum-exp, k best) into `records` (uint8)."""
        r = self._rows(shard_logits, params, history, history_len, mask, bias, id_offset=id_offset)
        rb = lib.mk_vp_record_bytes(k)
        assert records.dtype == torch.uint8 and records.numel() >= r.batch * rb and records.is_cuda
        check(lib.mk_sampler_vp_local(self._h, C.byref(r), k, records.data_ptr(), _stream_ptr(self.device)))
        return records

    def vp_merge(self, gathered: torch.Tensor, n_shards: int, batch: int, k: int, n_vocab_total: int, params, u):
        """Vocab-parallel step 2 on the all-gathered records [n_shards, batch, record_bytes]."""
        o = self._out(batch)
        c = params.to_c()
        check(lib.mk_sampler_vp_merge(self._h, gathered.data_ptr(), n_shards, batch, k, n_vocab_total, C.byref(c),
                                      _ptr(u), C.byref(o), _stream_ptr(self.device)))
        return self._result(batch)

    def sample_host(self, logits: np.ndarray, params: SamplingParams, u: np.ndarray, *, history=None, mask=None,
                    bias=None):
        """Host buffers in, host buffers out (copies inside): the form the reference's callers have."""
        assert logits.dtype == np.float32 and logits.ndim == 2 and logits.strides[1] == 4
        b, v = logits.shape
        r = RowsC()
        r.logits = logits.ctypes.data
        r.ld = logits.strides[0] // 4
        r.batch, r.n_vocab = b, v
        r.params = params.to_c()
        keep = [logits, u]
        if history is not None:
            assert history.dtype == np.int32 and history.ndim == 2
            r.history, r.history_ld, r.n_history = history.ctypes.data, history.strides[0] // 4, history.shape[1]
            keep.append(history)
        if mask is not None:
            assert mask.dtype == np.uint32 and mask.ndim == 2
            r.mask, r.mask_ld = mask.ctypes.data, mask.strides[0] // 4
            keep.append(mask)
        if bias is not None:
            assert bias.dtype == np.int32 and bias.ndim == 3 and bias.flags.c_contiguous
            r.bias, r.n_bias = bias.ctypes.data, bias.shape[1]
            keep.append(bias)
        tok = np.empty(b, dtype=np.int32)
        prob = np.empty(b, dtype=np.float32)
        flags = np.empty(b, dtype=np.uint32)
        o = SampleOutC()
        o.token, o.prob, o.flags = tok.ctypes.data, prob.ctypes.data, flags.ctypes.data
        check(lib.mk_sampler_sample_host(self._h, C.byref(r), u.ctypes.data if u is not None else None, C.byref(o)))
        return tok, prob, flags


def pack_bias(ids: np.ndarray, vals: np.ndarray) -> np.ndarray:
    """(ids int32 [B, nb], values float32 [B, nb]) -> int32 [B, nb, 2] in the layout of mk_bias."""
    out = np.empty(ids.shape + (2,), dtype=np.int32)
    out[..., 0] = ids
    out[..., 1] = vals.astype(np.float32).view(np.int32)
    return out


def pack_params(ps) -> np.ndarray:
    """List of SamplingParams -> int32 [B, 7] in the layout of mk_sampling_params (per-row parameters)."""
    out = np.empty((len(ps), 7), dtype=np.int32)
    for i, p in enumerate(ps):
        f = np.array([p.temperature, 0, p.top_p, p.min_p, p.presence_penalty, p.frequency_penalty,
                      p.repetition_penalty], dtype=np.float32).view(np.int32)
        out[i] = f
        out[i, 1] = np.array([p.top_k], dtype=np.uint32).view(np.int32)[0]
    return out
