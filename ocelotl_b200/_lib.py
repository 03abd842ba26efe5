"""ctypes binding of libocelotl_cuda.so (the C ABI in include/ocelotl_cuda.h).

The library is built in-tree by ocelotl_b200/build.py.  There is no fallback:
if it is missing, `load()` raises, so a GPU run can never silently take a CPU
path.
"""
from __future__ import annotations

import ctypes as C
import struct
from pathlib import Path

LIB_PATH = Path(__file__).resolve().parent / "libocelotl_cuda.so"

OCL_OK = 0
OCL_ERR_INVALID = -1
OCL_ERR_UNSUPPORTED = -2
OCL_ERR_CUDA = -3
OCL_ERR_OOM = -4
OCL_ERR_TIMEOUT = -5

_vp = C.c_void_p
_sz = C.c_size_t


class KvCacheDesc(C.Structure):
    """ocl_kv_cache"""
    _fields_ = [("k_dev", _vp), ("v_dev", _vp), ("dtype", C.c_int)] + [(n, _sz) for n in (
        "n_pages", "page_size", "n_kv_heads", "head_dim", "page_stride", "head_stride", "token_stride")]


# ocl_kv_rows as bytes (packing them costs a quarter of a Structure): positions, seqs, block table, n_seqs,
# max_pages, table_stride
KV_ROWS = struct.Struct("PPPNNN")


class LogitRulesDesc(C.Structure):
    """ocl_logit_rules"""
    _fields_ = [("history_dev", _vp), ("history_stride", _sz), ("history_max", _sz),
                ("history_lens_dev", _vp), ("prompt_lens_dev", _vp),
                ("repetition_dev", _vp), ("frequency_dev", _vp), ("presence_dev", _vp), ("bias_ids_dev", _vp),
                ("bias_values_dev", _vp), ("bias_stride", _sz), ("bias_count", _sz), ("allowed_dev", _vp), ("allowed_stride", _sz)]


# name -> (restype, argtypes); every symbol include/ocelotl_cuda.h declares.
SIGNATURES = {
    "ocl_cuda_init": (C.c_int, [C.c_int, C.POINTER(_vp)]),
    "ocl_cuda_destroy": (None, [_vp]),
    "ocl_last_error": (C.c_char_p, [_vp]),
    "ocl_set_stream": (C.c_int, [_vp, _vp]),
    "ocl_synchronize": (C.c_int, [_vp]),
    "ocl_set_pdl": (C.c_int, [_vp, C.c_int]),
    "ocl_set_gemm_min_rows": (C.c_int, [_vp, _sz]),
    "ocl_backend_id": (C.c_char_p, []),
    "ocl_abi_version": (C.c_int, []),
    "ocl_q_upload": (C.c_int, [_vp, C.c_int, _vp, _sz, _sz, C.c_int, C.POINTER(_vp)]),
    "ocl_q_upload_device": (C.c_int, [_vp, C.c_int, _vp, _sz, _sz, C.POINTER(_vp)]),
    "ocl_q_free": (C.c_int, [_vp]),
    "ocl_q_info": (C.c_int, [_vp, C.POINTER(C.c_int), C.POINTER(_sz), C.POINTER(_sz), C.POINTER(_sz)]),
    "ocl_q_device_ptr": (_vp, [_vp]),
    "ocl_q_dequant": (C.c_int, [_vp, _vp, _vp]),
    "ocl_q_download_gguf": (C.c_int, [_vp, _vp, _vp]),
    "ocl_q_linear": (C.c_int, [_vp, _vp, _vp, _sz, _sz, _sz, _vp, _vp]),
    "ocl_q_linear_noalloc": (C.c_int, [C.c_int, _vp, _sz, _sz, _vp, _sz, _vp, _vp, _vp]),
    "ocl_tp_comm_create": (C.c_int, [_vp, C.c_int, C.c_int, _sz, _sz, C.POINTER(_vp), _vp]),
    "ocl_tp_comm_open": (C.c_int, [_vp, _vp, _vp]),
    "ocl_tp_comm_destroy": (C.c_int, [_vp]),
    "ocl_tp_comm_packets": (_vp, [_vp]),
    "ocl_noalloc_take_device_errors": (C.c_int, [_vp, C.POINTER(C.c_uint)]),
    "ocl_q_linear_allreduce": (C.c_int, [_vp, _vp, _vp, _vp, _sz, _sz, _sz, _vp, _vp]),
    "ocl_q_linear_host": (C.c_int, [_vp, _vp, _vp, _sz, _sz, _sz, _vp, _vp]),
    "ocl_q_gemm_bf16": (C.c_int, [_vp, _vp, _vp, _sz, _sz, _sz, _vp]),
    "ocl_q_pair_gated": (C.c_int, [_vp, _vp, _vp, C.POINTER(_vp)]),
    "ocl_q_linear_gated": (C.c_int, [_vp, _vp, _vp, _sz, _sz, _sz, _vp]),
    "ocl_q_mlp_gated_silu": (C.c_int, [_vp, _vp, _vp, _vp, _sz, _sz, _sz, _vp, _vp]),
    "ocl_q_gemm_gated_bf16": (C.c_int, [_vp, _vp, _vp, _sz, _sz, _sz, _vp]),
    "ocl_argmax_f32": (C.c_int, [_vp, _vp, _sz, _sz, _vp]),
    "ocl_q_embed_rows": (C.c_int, [_vp, _vp, _vp, _sz, _vp]),
    "ocl_rope_create": (C.c_int, [_vp, _sz, C.c_double, _vp, C.c_int, C.POINTER(_vp)]),
    "ocl_rope_free": (C.c_int, [_vp]),
    "ocl_qk_norm_rope": (C.c_int, [_vp, _vp, _sz, _sz, _sz, C.POINTER(KvCacheDesc), C.c_char_p, _vp, _vp,
                                   C.c_float, _vp, _vp]),
    "ocl_paged_attention": (C.c_int, [_vp, _vp, _sz, _sz, _sz, C.POINTER(KvCacheDesc), C.c_char_p, C.c_float,
                                      _vp]),
    "ocl_logits_process": (C.c_int, [_vp, _vp, _sz, _sz, _sz, C.POINTER(LogitRulesDesc), _vp, _sz, _vp]),
    "ocl_take_device_errors": (C.c_int, [_vp, C.POINTER(C.c_uint), C.POINTER(C.c_uint)]),
}

_lib = None


def load() -> C.CDLL:
    """Load the library (once) and attach signatures.  Raises if it is absent."""
    global _lib
    if _lib is None:
        if not LIB_PATH.exists():
            raise RuntimeError(
                f"{LIB_PATH} is missing: build it with `python -m ocelotl_b200.build` "
                "(the quantized path has no CPU fallback)")
        lib = C.CDLL(str(LIB_PATH))
        for name, (res, args) in SIGNATURES.items():
            fn = getattr(lib, name)
            fn.restype = res
            fn.argtypes = args
        _lib = lib
    return _lib
