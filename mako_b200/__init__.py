"""mako_b200: the token-sampling path of jhanssen/mako as sm_100a CUDA kernels behind a C ABI.

The first use of any name below loads libmako_b200.so; that raises ImportError with the build command if the library
has not been built (`python -m mako_b200.build`, which itself needs no built library). Nothing here computes on the
CPU.
"""
_SAMPLER = {"BatchSampler", "KvCache", "KvPlan", "SampleResult", "SpecVerifyResult", "Sampler", "SamplingParams", "TokenLogprobs", "check_sampling", "pack_bias", "pack_params"}
_LIB = {"MakoError", "lib", "FLAG_ALL_MASKED", "FLAG_GUARD_BAND", "FLAG_NEAR_CDF_BOUNDARY", "FLAG_NO_CANDIDATE",
        "FLAG_OVERFLOW", "FLAG_TIMEOUT", "FLAG_HISTORY_FULL", "FLAG_VP_TRUNCATED", "FLAG_PLAN_INVALID", "FLAG_NO_ROOM",
        "FLAG_NO_PAGES"}
__all__ = sorted(_SAMPLER | _LIB | {"version", "synth"})


def __getattr__(name):
    import importlib
    if name in _SAMPLER:
        value = getattr(importlib.import_module(".sampler", __name__), name)
    elif name in _LIB:
        value = getattr(importlib.import_module("._lib", __name__), name)
    elif name in ("synth", "sampler", "build", "_lib"):
        value = importlib.import_module("." + name, __name__)
    else:
        raise AttributeError(f"module {__name__!r} has no attribute {name!r}")
    globals()[name] = value  # found without this function from now on
    return value


def version() -> str:
    from ._lib import lib
    return lib.mk_version().decode()
