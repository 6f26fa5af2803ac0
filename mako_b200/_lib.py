"""ctypes binding of libmako_b200.so (the C ABI declared in include/mako_b200.h).

The library is the product; there is no Python or CPU implementation behind these names. If the shared object is
missing the import fails with the build command to run, and every call fails when no CUDA device is present.
"""
from __future__ import annotations

import ctypes as C
import os

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.environ.get("MAKO_B200_LIB") or os.path.join(HERE, "libmako_b200.so")

MK_OK = 0
MK_ERR_INVALID_ARGUMENT = 1
MK_ERR_CUDA = 2
MK_ERR_UNSUPPORTED = 3
MK_ERR_NO_DEVICE = 4

FLAG_NEAR_CDF_BOUNDARY = 0x001
FLAG_GUARD_BAND = 0x002
FLAG_NO_CANDIDATE = 0x004
FLAG_ALL_MASKED = 0x008
FLAG_OVERFLOW = 0x010
FLAG_VP_TRUNCATED = 0x020
FLAG_TIMEOUT = 0x040
FLAG_HISTORY_FULL = 0x100
FLAG_PLAN_INVALID = 0x200
FLAG_NO_ROOM = 0x400
FLAG_NO_PAGES = 0x800

FP32, BF16, FP16 = 0, 1, 2

OVERLAP_OFF, OVERLAP_LAUNCH, OVERLAP_STABLE_SIDE_INPUTS = 0, 1, 2


class SamplingParamsC(C.Structure):
    _fields_ = [
        ("temperature", C.c_float),
        ("top_k", C.c_uint32),
        ("top_p", C.c_float),
        ("min_p", C.c_float),
        ("presence_penalty", C.c_float),
        ("frequency_penalty", C.c_float),
        ("repetition_penalty", C.c_float),
    ]


class RowsC(C.Structure):
    _fields_ = [
        ("logits", C.c_void_p),
        ("ld", C.c_uint64),
        ("batch", C.c_uint32),
        ("n_vocab", C.c_uint32),
        ("id_offset", C.c_int32),
        ("n_history", C.c_uint32),
        ("history", C.c_void_p),
        ("history_ld", C.c_uint64),
        ("history_len", C.c_void_p),
        ("mask", C.c_void_p),
        ("mask_ld", C.c_uint64),
        ("bias", C.c_void_p),
        ("n_bias", C.c_uint32),
        ("params_dev", C.c_void_p),
        ("params", SamplingParamsC),
    ]


class SampleOutC(C.Structure):
    _fields_ = [
        ("token", C.c_void_p),
        ("prob", C.c_void_p),
        ("flags", C.c_void_p),
        ("n_cand", C.c_void_p),
        ("cand_ids", C.c_void_p),
        ("cand_q", C.c_void_p),
        ("cand_cap", C.c_uint32),
    ]


class HeadC(C.Structure):
    _fields_ = [
        ("weight", C.c_void_p),
        ("down", C.c_void_p),
        ("up", C.c_void_p),
        ("scale", C.c_void_p),
        ("n_vocab", C.c_uint32),
        ("dim", C.c_uint32),
        ("n_adapters", C.c_uint32),
        ("rank", C.c_uint32),
        ("type", C.c_int),
    ]


class SpecRowsC(C.Structure):
    _fields_ = [
        ("logits", C.c_void_p),
        ("ld", C.c_uint64),
        ("draft_logits", C.c_void_p),
        ("draft_ld", C.c_uint64),
        ("type", C.c_int),
        ("n_seq", C.c_uint32),
        ("n_pos", C.c_uint32),
        ("n_vocab", C.c_uint32),
        ("drafts", C.c_void_p),
        ("u", C.c_void_p),
        ("temperature", C.c_void_p),
        ("draft_temperature", C.c_void_p),
        ("temperature_all", C.c_float),
        ("mask", C.c_void_p),
        ("mask_ld", C.c_uint64),
        ("mask_drafts", C.c_int),
    ]


class KvPagesC(C.Structure):
    _fields_ = [
        ("block_table", C.c_void_p),
        ("table_ld", C.c_uint64),
        ("table_cols", C.c_uint32),
        ("n_pages", C.c_void_p),
        ("free_list", C.c_void_p),
        ("free_cap", C.c_uint32),
        ("n_free", C.c_void_p),
        ("page_size", C.c_uint32),
    ]


class KvPlanC(C.Structure):
    _fields_ = [
        ("query_start", C.c_void_p),
        ("kv_len", C.c_void_p),
        ("positions", C.c_void_p),
        ("slots", C.c_void_p),
        ("token_seq", C.c_void_p),
        ("flags", C.c_void_p),
        ("max_tokens", C.c_uint32),
    ]


class LogprobRowsC(C.Structure):
    _fields_ = [
        ("logits", C.c_void_p),
        ("ld", C.c_uint64),
        ("type", C.c_int),
        ("rows", C.c_uint32),
        ("n_vocab", C.c_uint32),
        ("tokens", C.c_void_p),
        ("n_given", C.c_uint32),
        ("n_top", C.c_uint32),
        ("temperature", C.c_void_p),
        ("temperature_all", C.c_float),
        ("mask", C.c_void_p),
        ("mask_ld", C.c_uint64),
    ]


class KvCacheC(C.Structure):
    _fields_ = [
        ("k", C.c_void_p),
        ("v", C.c_void_p),
        ("k_scale", C.c_void_p),
        ("v_scale", C.c_void_p),
        ("page_stride", C.c_uint64),
        ("head_stride", C.c_uint64),
        ("token_stride", C.c_uint64),
        ("n_pages", C.c_uint32),
        ("n_heads", C.c_uint32),
        ("page_size", C.c_uint32),
        ("dim", C.c_uint32),
    ]


class KvRowsC(C.Structure):
    _fields_ = [
        ("k", C.c_void_p),
        ("v", C.c_void_p),
        ("k_ld", C.c_uint64),
        ("v_ld", C.c_uint64),
        ("q", C.c_void_p),
        ("q_out", C.c_void_p),
        ("q_ld", C.c_uint64),
        ("q_out_ld", C.c_uint64),
        ("n_q_heads", C.c_uint32),
        ("type", C.c_int),
        ("n_tokens", C.c_uint32),
        ("positions", C.c_void_p),
        ("slots", C.c_void_p),
    ]


class RotaryC(C.Structure):
    _fields_ = [
        ("inv_freq", C.c_void_p),
        ("dim", C.c_uint32),
        ("interleaved", C.c_int),
        ("scale", C.c_float),
    ]


class KvQueriesC(C.Structure):
    _fields_ = [
        ("q", C.c_void_p),
        ("out", C.c_void_p),
        ("q_ld", C.c_uint64),
        ("out_ld", C.c_uint64),
        ("n_q_heads", C.c_uint32),
        ("type", C.c_int),
        ("n_tokens", C.c_uint32),
        ("block_table", C.c_void_p),
        ("table_ld", C.c_uint64),
        ("table_cols", C.c_uint32),
        ("query_start", C.c_void_p),
        ("kv_len", C.c_void_p),
        ("n_seq", C.c_uint32),
        ("max_new", C.c_uint32),
        ("scale", C.c_float),
        ("window", C.c_uint32),
        ("workspace", C.c_void_p),
        ("workspace_bytes", C.c_uint64),
    ]


class MakoError(RuntimeError):
    def __init__(self, code: int, message: str):
        super().__init__(f"mako_b200 error {code}: {message}")
        self.code = code


def _load() -> C.CDLL:
    if not os.path.exists(LIB_PATH):
        raise ImportError(
            f"{LIB_PATH} is missing: build it with `python -m mako_b200.build` "
            "(nvcc, sm_100a). There is no fallback implementation."
        )
    try:  # libcudart comes with torch's CUDA wheels; loading torch first makes it resolvable
        import torch  # noqa: F401
    except Exception:
        pass
    lib = C.CDLL(LIB_PATH)
    vp = C.c_void_p
    lib.mk_version.restype = C.c_char_p
    lib.mk_last_error.restype = C.c_char_p
    lib.mk_row_bytes.restype = C.c_uint64
    lib.mk_row_bytes.argtypes = [C.c_uint32, C.c_uint32, C.c_int, C.c_uint32, C.c_uint32]
    lib.mk_check_sampling.argtypes = [C.POINTER(SamplingParamsC)]
    lib.mk_sampler_create.argtypes = [C.POINTER(vp), C.c_int, C.c_uint32, C.c_uint32]
    lib.mk_sampler_destroy.argtypes = [vp]
    lib.mk_sampler_destroy.restype = None
    lib.mk_sampler_sample_batch.argtypes = [vp, C.POINTER(RowsC), vp, C.POINTER(SampleOutC), vp]
    lib.mk_sample_rows_static.argtypes = [C.c_int, C.POINTER(RowsC), vp, C.POINTER(SampleOutC), vp]
    lib.mk_sampler_verify_batch.argtypes = [vp, C.POINTER(RowsC), vp, vp, vp, C.POINTER(SampleOutC), vp, vp]
    lib.mk_sampler_verify_pq_batch.argtypes = [vp, C.POINTER(RowsC), vp, C.c_uint64, vp, vp, vp, vp, vp, vp, vp, vp]
    lib.mk_spec_resolve.argtypes = [vp, C.c_uint32, C.c_uint32, vp, vp, vp, vp, vp]
    lib.mk_sampler_spec_round.argtypes = [vp, C.POINTER(RowsC), C.c_uint32, vp, vp, vp, C.POINTER(SampleOutC), vp, vp,
                                          vp, vp]
    lib.mk_spec_commit.argtypes = [vp, C.c_uint32, C.c_uint32, vp, vp, vp, vp, C.c_uint64, C.c_uint32, vp, vp, vp, vp]
    lib.mk_draft_pick.argtypes = [vp, vp, C.c_uint64, vp, vp, vp, C.c_uint64, vp, vp, C.c_uint32, C.c_uint32, C.c_uint32,
                                  C.c_uint32, C.c_uint32, vp, vp, vp]
    lib.mk_draft_pick_plain.argtypes = [vp, vp, C.c_uint64, C.c_uint32, C.c_uint32, vp, C.c_uint64, vp, C.c_uint32,
                                        C.c_float, vp, vp, vp, vp]
    lib.mk_rank_force.argtypes = [vp, vp, C.c_uint64, C.c_uint32, C.c_uint32, vp, C.c_uint32, vp, vp, vp]
    lib.mk_decode_commit.argtypes = [vp, C.c_uint32, vp, vp, vp, C.c_uint64, C.c_uint32, vp, vp, vp, vp, vp]
    lib.mk_head_logits.argtypes = [vp, C.POINTER(HeadC), vp, C.c_uint64, vp, C.c_uint32, vp, C.c_uint64, vp]
    lib.mk_spec_verify.argtypes = [vp, C.POINTER(SpecRowsC), vp, vp, vp, vp, vp, vp]
    lib.mk_kv_plan_step.argtypes = [vp, C.POINTER(KvPagesC), vp, vp, C.c_uint32, C.POINTER(KvPlanC), vp]
    lib.mk_token_logprobs.argtypes = [vp, C.POINTER(LogprobRowsC), vp, vp, vp, vp, vp, vp]
    lib.mk_kv_append.argtypes = [vp, C.POINTER(KvCacheC), C.POINTER(KvRowsC), C.POINTER(RotaryC), vp]
    lib.mk_kv_attention_bytes.restype = C.c_uint64
    lib.mk_kv_attention_bytes.argtypes = [C.POINTER(KvCacheC), C.POINTER(KvQueriesC)]
    lib.mk_kv_attention.argtypes = [vp, C.POINTER(KvCacheC), C.POINTER(KvQueriesC), vp]
    lib.mk_vp_record_bytes.restype = C.c_uint32
    lib.mk_vp_record_bytes.argtypes = [C.c_uint32]
    lib.mk_sampler_vp_local.argtypes = [vp, C.POINTER(RowsC), C.c_uint32, vp, vp]
    lib.mk_sampler_vp_merge.argtypes = [vp, vp, C.c_uint32, C.c_uint32, C.c_uint32, C.c_uint32,
                                        C.POINTER(SamplingParamsC), vp, C.POINTER(SampleOutC), vp]
    lib.mk_sampler_sample_host.argtypes = [vp, C.POINTER(RowsC), vp, C.POINTER(SampleOutC)]
    lib.mk_row_sampler_create.argtypes = [C.POINTER(vp), C.POINTER(SamplingParamsC), C.c_uint32, C.c_uint64, C.c_int]
    lib.mk_row_sampler_destroy.argtypes = [vp]
    lib.mk_row_sampler_destroy.restype = None
    lib.mk_row_sampler_greedy.argtypes = [vp]
    lib.mk_row_sampler_accept.argtypes = [vp, C.c_int32]
    lib.mk_row_sampler_sample.argtypes = [vp, vp, C.POINTER(C.c_int32)]
    lib.mk_row_sampler_verify.argtypes = [vp, vp, C.c_int32, C.POINTER(C.c_int32), C.POINTER(C.c_int32)]
    lib.mk_debug_expf.argtypes = [vp, vp, C.c_uint64, vp]
    lib.mk_debug_set_timing.argtypes = [vp, vp]
    lib.mk_sampler_set_overlap.argtypes = [vp, C.c_int]
    lib.mk_sampler_set_split.argtypes = [vp, C.c_int]
    lib.mk_debug_withhold_tile.argtypes = [vp, C.c_int, C.c_uint32]
    return lib


lib = _load()


def check(rc: int) -> None:
    if rc != MK_OK:
        raise MakoError(rc, lib.mk_last_error().decode())
