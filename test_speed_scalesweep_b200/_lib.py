"""ctypes binding of ``libscalesweep_b200.so`` (the C ABI in include/scalesweep_b200.h).

There is no fallback: if the library is missing or the tensors are not on a
CUDA device, calls raise.  Build the library with
``python -m test_speed_scalesweep_b200.build``.
"""
from __future__ import annotations

import ctypes
import os
import threading

import torch

from . import build as _build

_c_p = ctypes.c_void_p
_i64 = ctypes.c_int64
_int = ctypes.c_int
_f32 = ctypes.c_float

_SIGNATURES = {
    "ssw_abi_version": (_int, []),
    "ssw_status_string": (ctypes.c_char_p, [_int]),
    "ssw_last_error": (ctypes.c_char_p, []),
    "ssw_scalesweep_mse_nvfp4_quant_out": (_int, [_c_p, _int, _i64, _i64, _i64, _c_p, _c_p, _c_p, _int, _c_p]),
    "ssw_scalesweep_mse128_nvfp4_quant_out": (_int, [_c_p, _int, _i64, _i64, _i64, _c_p, _c_p, _c_p, _int, _c_p]),
    "ssw_scalesweep_mse_reference_nvfp4_quant_out": (_int, [_c_p, _int, _i64, _i64, _i64, _c_p, _c_p, _c_p, _int, _c_p]),
    "ssw_scalesweep_nvfp4_quant_out": (_int, [_c_p, _int, _i64, _i64, _i64, _c_p, _c_p, _c_p, _int, _c_p]),
    "ssw_scalesweep128_nvfp4_quant_out": (_int, [_c_p, _int, _i64, _i64, _i64, _c_p, _c_p, _c_p, _int, _c_p]),
    "ssw_rtn_nvfp4_quant_out": (_int, [_c_p, _int, _i64, _i64, _i64, _c_p, _c_p, _c_p, _int, _c_p]),
    "ssw_silu_and_mul": (_int, [_c_p, _int, _i64, _i64, _c_p, _c_p]),
    "ssw_rms_norm_scalesweep_mse_nvfp4_quant_out": (_int, [_c_p, _c_p, _c_p, _f32, _i64, _i64, _c_p,
                                                           _c_p, _c_p, _int, _c_p, _c_p]),
    "ssw_silu_and_mul_scalesweep_mse_nvfp4_quant_out": (_int, [_c_p, _int, _i64, _i64, _c_p, _c_p,
                                                               _c_p, _int, _c_p]),
    "ssw_absmax_workspace_bytes": (_i64, []),
    "ssw_absmax": (_int, [_c_p, _int, _i64, _c_p, _c_p, _c_p]),
    "ssw_global_scale_from_amax": (_int, [_c_p, _f32, _c_p, _c_p]),
    "ssw_global_scale_inv": (_int, [_c_p, _int, _i64, _f32, _c_p, _c_p, _c_p, _c_p]),
    "ssw_nvfp4_gemm_workspace_bytes": (_i64, [_i64, _i64, _i64]),
    "ssw_nvfp4_quant_gemm_workspace_bytes": (_i64, [_i64, _i64, _i64]),
    "ssw_nvfp4_quant_gemm": (_int, [_c_p, _int, _c_p, _c_p, _c_p, _c_p, _c_p, _i64, _i64, _i64,
                                    _c_p, _i64, _c_p, _c_p]),
    "ssw_nvfp4_gemm": (_int, [_c_p, _c_p, _c_p, _c_p, _c_p, _c_p, _i64, _i64, _i64, _c_p, _i64,
                              _c_p, _c_p]),
    "ssw_nvfp4_gemm_dependent": (_int, [_c_p, _c_p, _c_p, _c_p, _c_p, _c_p, _i64, _i64, _i64,
                                        _c_p, _i64, _c_p, _c_p]),
    "ssw_nvfp4_mma_rate_probe": (_int, [_int, _int, _c_p, _c_p, _c_p]),
    "ssw_global_scale_inv_noalloc_max_numel": (_i64, []),
    "ssw_global_scale_inv_noalloc": (_int, [_c_p, _int, _i64, _f32, _c_p, _c_p, _c_p]),
    "ssw_rotary_scalesweep_mse_nvfp4_kv_write": (_int, [_c_p, _int, _i64, _int, _c_p, _c_p, _c_p, _c_p,
                                                        _c_p, _c_p, _i64, _int, _int, _c_p, _c_p]),
    "ssw_nvfp4_kv_gather": (_int, [_c_p, _int, _i64, _c_p, _c_p, _c_p, _c_p]),
    "ssw_kv_pages_workspace_bytes": (_i64, [_i64, _i64, _int, _i64]),
    "ssw_kv_pages_fork": (_int, [_c_p, _c_p, _i64, _c_p, _c_p, _c_p, _i64, _c_p]),
    "ssw_kv_pages_free": (_int, [_c_p, _i64, _c_p, _c_p]),
    "ssw_kv_pages_extend": (_int, [_c_p, _i64, _c_p, _c_p, _i64, _c_p, _c_p, _i64, _c_p]),
    "ssw_kv_pages_compact": (_int, [_c_p, _c_p, _c_p, _i64, _c_p]),
    "ssw_kv_pages_copy": (_int, [_c_p, _i64, _c_p, _c_p, _c_p]),
    "ssw_nvfp4_paged_attention_workspace_bytes": (_i64, [_c_p, _c_p, _int]),
    "ssw_nvfp4_paged_attention": (_int, [_c_p, _c_p, _int, _c_p, _c_p, _c_p, _i64, _c_p]),
}


class KVCache(ctypes.Structure):
    """``ssw_kv_cache``."""
    _fields_ = [("codes", _c_p), ("scales", _c_p), ("codes_page_stride", _i64),
                ("scales_page_stride", _i64), ("input_scale", _c_p), ("num_pages", _i64),
                ("page_size", ctypes.c_int32), ("kv_heads", ctypes.c_int32),
                ("head_size", ctypes.c_int32)]


class KVHeads(ctypes.Structure):
    """``ssw_kv_heads``."""
    _fields_ = [("data", _c_p), ("token_stride", _i64), ("head_stride", _i64)]


class KVAttention(ctypes.Structure):
    """``ssw_kv_attention``."""
    _fields_ = [("block_table", _c_p), ("block_table_stride", _i64), ("seq_lens", _c_p),
                ("query_start", _c_p), ("lse", _c_p), ("status", _c_p), ("tokens", _i64),
                ("seqs", ctypes.c_int32), ("block_table_columns", ctypes.c_int32),
                ("q_heads", ctypes.c_int32), ("max_query_len", ctypes.c_int32),
                ("max_seq_len", ctypes.c_int32), ("causal", ctypes.c_int32),
                ("window", ctypes.c_int32), ("softmax_scale", _f32)]


class KVPages(ctypes.Structure):
    """``ssw_kv_pages``."""
    _fields_ = [("refcount", _c_p), ("block_table", _c_p), ("table_stride", _i64),
                ("seq_lens", _c_p), ("status", _c_p), ("num_pages", ctypes.c_int32),
                ("max_seqs", ctypes.c_int32), ("columns", ctypes.c_int32),
                ("page_size", ctypes.c_int32)]


class KVPool(ctypes.Structure):
    """``ssw_kv_pool``."""
    _fields_ = [("codes", _c_p), ("scales", _c_p), ("codes_layer_stride", _i64),
                ("scales_layer_stride", _i64), ("codes_page_stride", _i64),
                ("scales_page_stride", _i64), ("codes_page_bytes", _i64),
                ("scales_page_bytes", _i64), ("num_pages", _i64), ("layers", ctypes.c_int32)]


ABI_VERSION = 1
SSW_OK, SSW_ERR_INVALID_ARGUMENT, SSW_ERR_UNSUPPORTED, SSW_ERR_CUDA, SSW_ERR_TIMEOUT = range(5)

_lock = threading.Lock()
_handle = None


def library_path() -> str:
    return _build.LIB_PATH


def lib() -> ctypes.CDLL:
    """Load the CUDA library (once).  Raises if it has not been built."""
    global _handle
    if _handle is not None:
        return _handle
    with _lock:
        if _handle is None:
            path = library_path()
            if not os.path.exists(path):
                raise RuntimeError(
                    f"{path} is missing: the scale-sweep CUDA library must be built "
                    "(python -m test_speed_scalesweep_b200.build); there is no CPU fallback")
            h = ctypes.CDLL(path)
            for name, (res, args) in _SIGNATURES.items():
                fn = getattr(h, name)
                fn.restype = res
                fn.argtypes = args
            if h.ssw_abi_version() != ABI_VERSION:
                raise RuntimeError("libscalesweep_b200.so ABI version mismatch; rebuild it")
            _handle = h
    return _handle


def check(status: int) -> None:
    if status == SSW_OK:
        return
    h = lib()
    msg = (h.ssw_last_error() or b"").decode() or h.ssw_status_string(status).decode()
    if status == SSW_ERR_INVALID_ARGUMENT:
        raise ValueError(msg)
    if status == SSW_ERR_UNSUPPORTED:
        raise NotImplementedError(msg)
    if status == SSW_ERR_TIMEOUT:
        raise TimeoutError(msg)
    raise RuntimeError(msg)


DTYPE_CODES = {torch.bfloat16: 0, torch.float16: 1}


def dtype_code(t: torch.Tensor) -> int:
    try:
        return DTYPE_CODES[t.dtype]
    except KeyError:
        raise ValueError(f"input dtype must be torch.bfloat16 or torch.float16, got {t.dtype}") from None


def stream_handle(device: torch.device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


_kv = None


def kv_binding():
    """The native binding of the KV-cache operators (``_kv_binding.so``)."""
    global _kv
    if _kv is None:
        lib()  # the library it links to: the same checks, the same error
        if not os.path.exists(_build.BINDING_PATH):
            raise RuntimeError(
                f"{_build.BINDING_PATH} is missing: it is built with the CUDA library "
                "(python -m test_speed_scalesweep_b200.build); there is no fallback")
        from . import _kv_binding
        _kv = _kv_binding
    return _kv
