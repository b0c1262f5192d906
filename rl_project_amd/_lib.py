"""ctypes binding of libflsampler.so (include/fl_sampler.h).

The library is loaded once, after ``torch`` (torch's HIP runtime is the one
the library binds to, so device pointers and streams are shared).  There is
no fallback: if the library is missing or fails to load, every sampling call
raises ``SamplerLibraryError``.
"""

from __future__ import annotations

import ctypes
import os
from typing import Optional

import torch  # noqa: F401  (loads the HIP runtime the library binds to)

# FL_SAMPLER_LIB names another build of the library (the host-sanitizer build).
LIB_PATH = os.environ.get("FL_SAMPLER_LIB") or os.path.join(os.path.dirname(os.path.abspath(__file__)), "_lib",
                                                            "libflsampler.so")

FL_ABI_VERSION = 8
FL_DTYPE_F32, FL_DTYPE_BF16, FL_DTYPE_F16, FL_DTYPE_E4M3 = 0, 1, 2, 3
FL_OK, FL_EIO, FL_EINVAL, FL_ENOTSUP = 0, -5, -22, -95
FL_ROW_OK, FL_ROW_NAN, FL_ROW_INF, FL_ROW_BAD_HISTORY, FL_ROW_LIMIT, FL_ROW_ALL_MASKED = 0, 1, 2, 4, 8, 16
FL_FLAG_NO_SELECT = 1
FL_FLAG_APPEND_HISTORY = 2
FL_FLAG_EXACT_COUNTS = 4
FL_FLAG_ONLY_LIMITED = 8
FL_MAX_VOCAB_F32 = 262144
FL_MAX_VOCAB_16 = 262144
FL_SPEC_STATIC_MAX_BATCH = 4096
FL_MAX_HISTORY = 65536

ROW_STATUS_NAMES = {
    FL_ROW_NAN: "NaN logit",
    FL_ROW_INF: "+inf logit after scaling",
    FL_ROW_BAD_HISTORY: "history id outside [0, vocab)",
    FL_ROW_LIMIT: "row exceeds an internal capacity",
    FL_ROW_ALL_MASKED: "every logit filtered out",
}

_p = ctypes.c_void_p


class SampleArgs(ctypes.Structure):
    _fields_ = [
        ("struct_size", ctypes.c_uint32), ("dtype", ctypes.c_int32),
        ("logits", _p), ("batch", ctypes.c_int64), ("vocab", ctypes.c_int64), ("ld", ctypes.c_int64),
        ("temperature", _p), ("top_k", _p), ("top_p", _p), ("min_p", _p), ("rep_penalty", _p),
        ("softcap", ctypes.c_float), ("flags", ctypes.c_int32),
        ("hist_ids", _p), ("hist_ld", ctypes.c_int64), ("hist_len", _p),
        ("stop_ids", _p), ("stop_ld", ctypes.c_int64), ("n_stop", ctypes.c_int64),
        ("uniforms", _p), ("finished_in", _p),
        ("out_token", _p), ("out_finished", _p), ("out_status", _p), ("out_logprob", _p), ("out_desc", _p),
        ("uniform_div", ctypes.c_int64),
    ]


class RowValues(ctypes.Structure):
    _fields_ = [
        ("temperature", ctypes.c_float), ("top_k", ctypes.c_int32), ("top_p", ctypes.c_float),
        ("min_p", ctypes.c_float), ("rep_penalty", ctypes.c_float), ("hist_len", ctypes.c_int32),
    ]


class SpecArgs(ctypes.Structure):
    _fields_ = [
        ("struct_size", ctypes.c_uint32), ("dtype", ctypes.c_int32),
        ("target", _p), ("draft", _p),
        ("batch", ctypes.c_int64), ("k", ctypes.c_int64), ("vocab", ctypes.c_int64), ("ld", ctypes.c_int64),
        ("temperature", _p), ("softcap", ctypes.c_float),
        ("target_desc", _p), ("draft_desc", _p), ("draft_ids", _p), ("u_accept", _p), ("u_resample", _p),
        ("bonus_token", _p), ("out_n_accepted", _p), ("out_tokens", _p), ("out_ratio", _p),
        ("workspace", _p), ("workspace_bytes", ctypes.c_int64),
    ]


class RowStatsArgs(ctypes.Structure):
    _fields_ = [
        ("struct_size", ctypes.c_uint32), ("dtype", ctypes.c_int32),
        ("logits", _p), ("ref_logits", _p),
        ("rows", ctypes.c_int64), ("vocab", ctypes.c_int64), ("ld", ctypes.c_int64), ("ref_ld", ctypes.c_int64),
        ("labels", _p), ("ignore_index", ctypes.c_int64),
        ("out_logprob", _p), ("out_entropy", _p), ("out_kl", _p), ("out_lse", _p),
    ]


class LmHeadArgs(ctypes.Structure):
    _fields_ = [
        ("struct_size", ctypes.c_uint32), ("dtype", ctypes.c_int32),
        ("hidden", _p), ("weight", _p),
        ("batch", ctypes.c_int64), ("dim", ctypes.c_int64), ("vocab", ctypes.c_int64), ("ld_hidden", ctypes.c_int64),
        ("temperature", _p), ("top_k", _p), ("top_p", _p), ("min_p", _p), ("repetition_penalty", _p),
        ("hist_ids", _p), ("hist_len", _p), ("hist_ld", ctypes.c_int64), ("softcap", ctypes.c_float),
        ("uniforms", _p), ("out_token", _p), ("out_status", _p), ("out_logprob", _p), ("out_logits", _p),
        ("workspace", _p), ("workspace_bytes", ctypes.c_int64),
    ]


class ScoreArgs(ctypes.Structure):
    _fields_ = [
        ("struct_size", ctypes.c_uint32), ("dtype", ctypes.c_int32),
        ("logits", _p), ("rows", ctypes.c_int64), ("vocab", ctypes.c_int64), ("ld", ctypes.c_int64),
        ("tokens", _p), ("ignore_index", ctypes.c_int64), ("top_k", ctypes.c_int64),
        ("out_logprob", _p), ("out_entropy", _p), ("out_lse", _p), ("out_rank", _p),
        ("out_top_ids", _p), ("out_top_logprobs", _p), ("out_saved", _p),
        ("workspace", _p), ("workspace_bytes", ctypes.c_int64),
    ]


class ScoreGradArgs(ctypes.Structure):
    _fields_ = [
        ("struct_size", ctypes.c_uint32), ("dtype", ctypes.c_int32),
        ("logits", _p), ("rows", ctypes.c_int64), ("vocab", ctypes.c_int64), ("ld", ctypes.c_int64),
        ("tokens", _p), ("ignore_index", ctypes.c_int64), ("saved", _p),
        ("grad_logprob", _p), ("grad_entropy", _p), ("grad_lse", _p),
        ("out_grad", _p), ("out_ld", ctypes.c_int64),
    ]


class NormArgs(ctypes.Structure):
    _fields_ = [
        ("struct_size", ctypes.c_uint32), ("dtype", ctypes.c_int32), ("wdtype", ctypes.c_int32), ("eps", ctypes.c_float),
        ("x", _p), ("rows", ctypes.c_int64), ("dim", ctypes.c_int64), ("ld", ctypes.c_int64),
        ("weight", _p), ("bias", _p), ("out", _p), ("out_ld", ctypes.c_int64), ("out_mean", _p), ("out_rstd", _p),
    ]


class NormGradArgs(ctypes.Structure):
    _fields_ = [
        ("struct_size", ctypes.c_uint32), ("dtype", ctypes.c_int32), ("wdtype", ctypes.c_int32), ("reserved", ctypes.c_int32),
        ("x", _p), ("rows", ctypes.c_int64), ("dim", ctypes.c_int64), ("ld", ctypes.c_int64),
        ("weight", _p), ("grad", _p), ("grad_ld", ctypes.c_int64), ("mean", _p), ("rstd", _p),
        ("out_dx", _p), ("out_ld", ctypes.c_int64), ("out_dweight", _p), ("out_dbias", _p),
        ("workspace", _p), ("workspace_bytes", ctypes.c_int64),
    ]


class HeadArgs(ctypes.Structure):
    _fields_ = [
        ("struct_size", ctypes.c_uint32), ("dtype", ctypes.c_int32),
        ("hidden", _p), ("weight", _p), ("rows", ctypes.c_int64), ("dim", ctypes.c_int64), ("vocab", ctypes.c_int64),
        ("ld_hidden", ctypes.c_int64), ("tokens", _p), ("ignore_index", ctypes.c_int64),
        ("out_logprob", _p), ("out_entropy", _p), ("out_lse", _p), ("out_saved", _p),
        ("workspace", _p), ("workspace_bytes", ctypes.c_int64),
    ]


class HeadGradArgs(ctypes.Structure):
    _fields_ = [
        ("struct_size", ctypes.c_uint32), ("dtype", ctypes.c_int32),
        ("hidden", _p), ("weight", _p), ("rows", ctypes.c_int64), ("dim", ctypes.c_int64), ("vocab", ctypes.c_int64),
        ("ld_hidden", ctypes.c_int64), ("tokens", _p), ("ignore_index", ctypes.c_int64), ("saved", _p),
        ("grad_logprob", _p), ("grad_entropy", _p), ("grad_lse", _p), ("out_dhidden", _p), ("out_dweight", _p),
        ("workspace", _p), ("workspace_bytes", ctypes.c_int64),
    ]


class RopeArgs(ctypes.Structure):
    _fields_ = [
        ("struct_size", ctypes.c_uint32), ("dtype", ctypes.c_int32), ("wdtype", ctypes.c_int32), ("flags", ctypes.c_int32),
        ("q", _p), ("k", _p), ("tokens", ctypes.c_int64), ("heads", ctypes.c_int64), ("kv_heads", ctypes.c_int64),
        ("dim", ctypes.c_int64), ("rotated", ctypes.c_int64),
        ("q_ld", ctypes.c_int64), ("q_hs", ctypes.c_int64), ("k_ld", ctypes.c_int64), ("k_hs", ctypes.c_int64),
        ("positions", _p), ("inv_freq", _p), ("q_weight", _p), ("k_weight", _p),
        ("eps", ctypes.c_float), ("gain", ctypes.c_float), ("norm", ctypes.c_int32), ("reserved", ctypes.c_int32),
        ("out_q", _p), ("out_k", _p),
    ]


class RopeGradArgs(ctypes.Structure):
    _fields_ = [
        ("struct_size", ctypes.c_uint32), ("reserved", ctypes.c_int32), ("fwd", RopeArgs),
        ("grad_q", _p), ("grad_k", _p), ("out_dwq", _p), ("out_dwk", _p), ("workspace", _p), ("workspace_bytes", ctypes.c_int64),
    ]


class Cache(ctypes.Structure):
    _fields_ = [
        ("k", _p), ("v", _p), ("k_scale", _p), ("v_scale", _p),
        ("pages", ctypes.c_int64), ("heads", ctypes.c_int64), ("page_size", ctypes.c_int64), ("dim", ctypes.c_int64),
        ("dtype", ctypes.c_int32), ("reserved", ctypes.c_int32),
    ]


class CacheRows(ctypes.Structure):
    _fields_ = [
        ("table", _p), ("lengths", _p), ("starts", _p),
        ("seqs", ctypes.c_int64), ("tokens", ctypes.c_int64), ("table_width", ctypes.c_int64), ("table_ld", ctypes.c_int64),
    ]


class CacheArgs(ctypes.Structure):
    _fields_ = [
        ("struct_size", ctypes.c_uint32), ("dtype", ctypes.c_int32), ("cache", Cache), ("rows", CacheRows),
        ("k", _p), ("v", _p), ("k_ld", ctypes.c_int64), ("k_hs", ctypes.c_int64), ("v_ld", ctypes.c_int64), ("v_hs", ctypes.c_int64),
    ]


class AttnArgs(ctypes.Structure):
    _fields_ = [
        ("struct_size", ctypes.c_uint32), ("dtype", ctypes.c_int32), ("cache", Cache), ("rows", CacheRows),
        ("q", _p), ("q_heads", ctypes.c_int64), ("q_ld", ctypes.c_int64), ("q_hs", ctypes.c_int64),
        ("out", _p), ("out_ld", ctypes.c_int64), ("out_hs", ctypes.c_int64), ("out_lse", _p),
        ("scale", ctypes.c_float), ("softcap", ctypes.c_float), ("window", ctypes.c_int64), ("sinks", ctypes.c_int64),
        ("workspace", _p), ("workspace_bytes", ctypes.c_int64),
    ]


FL_ROPE_MAX_DIM = 512
FL_ROPE_INTERLEAVED, FL_ROPE_POSITIONS32 = 1, 2
FL_CACHE_MAX_DIM = 256
FL_HEAD_MAX_ROWS = 131072
FL_NORM_MAX_DIM = 16384
FL_SCORE_MAX_TOPK = 64
FL_LM_HEAD_MAX_BATCH = 64
FL_LM_HEAD_MAX_TOPK = 64
FL_LM_HEAD_MAX_CAND = 4096


# fl_row_desc: {float y_cut; int32 idx_cut; float shift; float inv_mass; double mass; int32 status; int32 n_kept}
ROW_DESC_BYTES = 32


class SamplerLibraryError(RuntimeError):
    """The HIP sampling library is missing, failed to load, or returned an error."""


_lib: Optional[ctypes.CDLL] = None


def lib() -> ctypes.CDLL:
    """Load libflsampler.so (once) and check its ABI version."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(LIB_PATH):
        raise SamplerLibraryError(
            f"{LIB_PATH} is missing: build it with `python -m rl_project_amd.build` "
            "(there is no CPU fallback)")
    try:
        handle = ctypes.CDLL(LIB_PATH)
    except OSError as exc:  # pragma: no cover - depends on the machine
        raise SamplerLibraryError(f"cannot load {LIB_PATH}: {exc}") from exc
    # (before any other symbol is bound: an older library may lack some)
    try:
        handle.fl_abi_version.restype = ctypes.c_int
        version = handle.fl_abi_version()
    except AttributeError:
        raise SamplerLibraryError(f"{LIB_PATH} has no fl_abi_version: not this library") from None
    if version != FL_ABI_VERSION:
        raise SamplerLibraryError(f"ABI version {version} of {LIB_PATH} != {FL_ABI_VERSION}: "
                                  "build it with `python -m rl_project_amd.build`")
    handle.fl_last_error.restype = ctypes.c_char_p
    handle.fl_sample.argtypes = [ctypes.POINTER(SampleArgs), _p]
    handle.fl_sample.restype = ctypes.c_int
    handle.fl_sample_exact.argtypes = [ctypes.POINTER(SampleArgs), _p]
    handle.fl_sample_exact.restype = ctypes.c_int
    handle.fl_fill_rows.argtypes = [ctypes.POINTER(RowValues), ctypes.c_int64, _p, _p]
    handle.fl_fill_rows.restype = ctypes.c_int
    handle.fl_apply_filter.argtypes = [ctypes.POINTER(SampleArgs), _p, _p, ctypes.c_int64, _p, _p, _p]
    handle.fl_apply_filter.restype = ctypes.c_int
    handle.fl_spec_verify.argtypes = [ctypes.POINTER(SpecArgs), _p]
    handle.fl_spec_verify.restype = ctypes.c_int
    handle.fl_spec_verify_static.argtypes = [ctypes.POINTER(SpecArgs), _p]
    handle.fl_spec_verify_static.restype = ctypes.c_int
    handle.fl_spec_workspace_bytes.argtypes = [ctypes.c_int64, ctypes.POINTER(ctypes.c_size_t)]
    handle.fl_spec_workspace_bytes.restype = ctypes.c_int
    handle.fl_spec_cache_workspace_bytes.argtypes = [ctypes.c_int64, ctypes.c_int64, ctypes.POINTER(ctypes.c_size_t)]
    handle.fl_spec_cache_workspace_bytes.restype = ctypes.c_int
    handle.fl_lm_head_sample.argtypes = [ctypes.POINTER(LmHeadArgs), _p]
    handle.fl_lm_head_sample.restype = ctypes.c_int
    handle.fl_lm_head_workspace_bytes.argtypes = [ctypes.c_int64, ctypes.c_int64, ctypes.POINTER(ctypes.c_size_t)]
    handle.fl_lm_head_workspace_bytes.restype = ctypes.c_int
    handle.fl_row_stats.argtypes = [ctypes.POINTER(RowStatsArgs), _p]
    handle.fl_row_stats.restype = ctypes.c_int
    handle.fl_score_tokens.argtypes = [ctypes.POINTER(ScoreArgs), _p]
    handle.fl_score_tokens.restype = ctypes.c_int
    handle.fl_score_workspace_bytes.argtypes = [ctypes.c_int64, ctypes.c_int64, ctypes.c_int64, ctypes.POINTER(ctypes.c_size_t)]
    handle.fl_score_workspace_bytes.restype = ctypes.c_int
    handle.fl_score_tokens_grad.argtypes = [ctypes.POINTER(ScoreGradArgs), _p]
    handle.fl_score_tokens_grad.restype = ctypes.c_int
    handle.fl_layer_norm.argtypes = [ctypes.POINTER(NormArgs), _p]
    handle.fl_layer_norm.restype = ctypes.c_int
    handle.fl_layer_norm_grad.argtypes = [ctypes.POINTER(NormGradArgs), _p]
    handle.fl_layer_norm_grad.restype = ctypes.c_int
    handle.fl_layer_norm_grad_workspace_bytes.argtypes = [ctypes.c_int64, ctypes.c_int64, ctypes.c_int32,
                                                          ctypes.POINTER(ctypes.c_size_t)]
    handle.fl_layer_norm_grad_workspace_bytes.restype = ctypes.c_int
    handle.fl_head_logprobs.argtypes = [ctypes.POINTER(HeadArgs), _p]
    handle.fl_head_logprobs.restype = ctypes.c_int
    handle.fl_head_workspace_bytes.argtypes = [ctypes.c_int64, ctypes.c_int64, ctypes.POINTER(ctypes.c_size_t)]
    handle.fl_head_workspace_bytes.restype = ctypes.c_int
    handle.fl_head_logprobs_grad.argtypes = [ctypes.POINTER(HeadGradArgs), _p]
    handle.fl_head_logprobs_grad.restype = ctypes.c_int
    handle.fl_head_grad_workspace_bytes.argtypes = [ctypes.c_int64, ctypes.c_int64, ctypes.c_int64, ctypes.c_int32,
                                                    ctypes.POINTER(ctypes.c_size_t)]
    handle.fl_head_grad_workspace_bytes.restype = ctypes.c_int
    for name, args in (("fl_qk_norm_rope", RopeArgs), ("fl_qk_norm_rope_grad", RopeGradArgs), ("fl_cache_write", CacheArgs),
                       ("fl_cache_read", CacheArgs), ("fl_paged_attention", AttnArgs)):
        getattr(handle, name).argtypes = [ctypes.POINTER(args), _p]
        getattr(handle, name).restype = ctypes.c_int
    handle.fl_qk_norm_rope_grad_workspace_bytes.argtypes = [ctypes.c_int64, ctypes.c_int64, ctypes.POINTER(ctypes.c_size_t)]
    handle.fl_qk_norm_rope_grad_workspace_bytes.restype = ctypes.c_int
    handle.fl_paged_attention_workspace_bytes.argtypes = [ctypes.POINTER(AttnArgs), ctypes.POINTER(ctypes.c_size_t)]
    handle.fl_paged_attention_workspace_bytes.restype = ctypes.c_int
    _lib = handle
    return handle


AUTOGRAD_PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "_lib", "_fl_autograd.so")
_AUTOGRAD_ENTRIES = ("fl_last_error", "fl_score_tokens", "fl_score_workspace_bytes", "fl_score_tokens_grad", "fl_layer_norm",
                     "fl_layer_norm_grad", "fl_layer_norm_grad_workspace_bytes", "fl_head_logprobs", "fl_head_workspace_bytes",
                     "fl_head_logprobs_grad", "fl_head_grad_workspace_bytes",
                     "fl_qk_norm_rope", "fl_qk_norm_rope_grad", "fl_qk_norm_rope_grad_workspace_bytes", "fl_cache_write",
                     "fl_cache_read", "fl_paged_attention", "fl_paged_attention_workspace_bytes")
_autograd = None


def autograd():
    """The extension that launches score_tokens, layer_norm, lm_head_logprobs,
    qk_norm_rope and the calls on a paged cache, and holds their autograd nodes (loaded once), bound to this library's entry points."""
    global _autograd
    if _autograd is not None:
        return _autograd
    handle = lib()
    if not os.path.exists(AUTOGRAD_PATH):
        raise SamplerLibraryError(f"{AUTOGRAD_PATH} is missing: build it with `python -m rl_project_amd.build`")
    from importlib.machinery import ExtensionFileLoader
    from importlib.util import module_from_spec, spec_from_file_location

    spec = spec_from_file_location("_fl_autograd", AUTOGRAD_PATH, loader=ExtensionFileLoader("_fl_autograd", AUTOGRAD_PATH))
    try:
        module = module_from_spec(spec)
        spec.loader.exec_module(module)
    except ImportError as exc:
        raise SamplerLibraryError(f"cannot load {AUTOGRAD_PATH}: {exc}") from exc
    module.bind([ctypes.cast(getattr(handle, n), ctypes.c_void_p).value for n in _AUTOGRAD_ENTRIES])
    _autograd = module
    return module


def check(rc: int, what: str) -> None:
    if rc != FL_OK:
        msg = lib().fl_last_error().decode(errors="replace")
        kind = {FL_EINVAL: ValueError, FL_ENOTSUP: NotImplementedError}.get(rc, SamplerLibraryError)
        raise kind(f"{what} failed ({rc}): {msg}")


def ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def stream_handle(device: torch.device) -> int:
    """The device's current stream (hipStream_t as an int), read at each
    launch: the raw query where torch has it (no Stream object built)."""
    if _raw_stream is not None:
        idx = device.index if device.index is not None else torch.cuda.current_device()
        return _raw_stream(idx)
    return torch.cuda.current_stream(device).cuda_stream


EXPORTED_SYMBOLS = ("fl_sample", "fl_sample_exact", "fl_fill_rows", "fl_apply_filter", "fl_spec_verify", "fl_spec_verify_static",
                    "fl_spec_workspace_bytes", "fl_spec_cache_workspace_bytes", "fl_lm_head_sample", "fl_lm_head_workspace_bytes", "fl_row_stats",
                    "fl_score_tokens", "fl_score_workspace_bytes", "fl_score_tokens_grad",
                    "fl_layer_norm", "fl_layer_norm_grad", "fl_layer_norm_grad_workspace_bytes",
                    "fl_head_logprobs", "fl_head_workspace_bytes", "fl_head_logprobs_grad", "fl_head_grad_workspace_bytes",
                    "fl_qk_norm_rope", "fl_qk_norm_rope_grad", "fl_qk_norm_rope_grad_workspace_bytes",
                    "fl_cache_write", "fl_cache_read", "fl_paged_attention", "fl_paged_attention_workspace_bytes",
                    "fl_last_error", "fl_abi_version")
