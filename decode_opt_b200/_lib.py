"""ctypes binding of ``libdecode_gemm_b200.so`` (include/decode_gemm_b200.h).

The library is the product; there is no fallback.  ``lib()`` raises when the
shared object is missing or cannot be loaded, so a GPU run without the built
extension fails loudly instead of computing anything elsewhere.
"""

from __future__ import annotations

import ctypes
import os

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "libdecode_gemm_b200.so")

ABI_VERSION = 10

LAYOUT_RAW = 0
LAYOUT_PACKED = 1
LAYOUT_PACKED_SWIZZLED = 2
GRID_CLUSTER = -2              # DG_GRID_CLUSTER

FLAG_INJECT_TIMEOUT = 2
FLAG_INDEPENDENT_INPUTS = 4
FLAG_SWAP_AB = 512              # DG_FLAG_SWAP_AB
STATIC_SEM_INTS = 4096          # DG_STATIC_SEM_INTS
STATIC_WS_FLOATS = 2097152      # DG_STATIC_WS_FLOATS

STATUS_OK = 0
ERR_INJECTED_TIMEOUT = 0x51

# Every symbol include/decode_gemm_b200.h declares.
EXPORTED_SYMBOLS = (
    "dg_abi_version", "dg_plan", "dg_make_weight_map", "dg_make_activation_map",
    "dg_launch_with_maps", "dg_launch", "dg_prepack_weight", "dg_padded_n",
    "dg_packed_weight_bytes", "dg_status_string", "dg_flush_l2", "dg_probe_bulk_stream",
    "dg_probe_naive_read", "dg_num_sms", "dg_launch_static_scratch", "dg_probe_mma",
    "dg_launch_gather", "dg_gather_wait", "dg_ipc_export", "dg_ipc_import", "dg_ipc_release",
    "dg_quantize_act", "dg_max_active_clusters", "dg_launch_quantized", "dg_launch_gather_lines",
    "dg_host_device_pointer", "dg_copy_from_host",
    # include/decode_attention_b200.h
    "dg_build_block_tables", "dg_rotary", "dg_paged_attention", "dg_attention_workspace_bytes",
)

# include/decode_attention_b200.h
TYPE_BF16, TYPE_FP16, TYPE_FP32, TYPE_E4M3 = 0, 1, 2, 3
PAIR_HALF, PAIR_ADJACENT = 0, 1
MAX_ROT = 512                   # DG_MAX_ROT
ERR_LENGTH, ERR_POOL, ERR_TABLE_WIDTH, ERR_TOKENS = 0xA1, 0xA2, 0xA3, 0xA4
ERR_POSITION, ERR_SLOT = 0xB1, 0xB2
ERR_PAGE, ERR_SEQ_LEN = 0xC1, 0xC2


class DgConfig(ctypes.Structure):
    _fields_ = [
        ("m_tile", ctypes.c_int),
        ("block_n", ctypes.c_int),
        ("subs", ctypes.c_int),
        ("stages", ctypes.c_int),
        ("layout", ctypes.c_int),
        ("pdl", ctypes.c_int),
        ("split_k", ctypes.c_int),
        ("grid_ctas", ctypes.c_int),
        ("epi_warps", ctypes.c_int),
        ("flags", ctypes.c_int),
        ("timeout_ns", ctypes.c_ulonglong),
        ("pack_rows", ctypes.c_int),
    ]


class DgProblem(ctypes.Structure):
    _fields_ = [
        ("M", ctypes.c_int),
        ("N", ctypes.c_int),
        ("K", ctypes.c_int),
        ("activation", ctypes.c_void_p),
        ("weight", ctypes.c_void_p),
        ("weight_scales", ctypes.c_void_p),
        ("activation_scales", ctypes.c_void_p),
        ("output", ctypes.c_void_p),
        ("splitk_ws", ctypes.c_void_p),
        ("splitk_sem", ctypes.c_void_p),
        ("status", ctypes.c_void_p),
    ]


class DgPlanInfo(ctypes.Structure):
    _fields_ = [
        ("grid_x", ctypes.c_uint),
        ("grid_y", ctypes.c_uint),
        ("grid_z", ctypes.c_uint),
        ("block_x", ctypes.c_uint),
        ("smem_bytes", ctypes.c_uint),
        ("num_output_tiles", ctypes.c_int),
        ("padded_n", ctypes.c_int),
        ("stages", ctypes.c_int),
        ("n_mma", ctypes.c_int),
        ("a_rows", ctypes.c_int),
        ("mma_m", ctypes.c_int),
        ("epi_warps", ctypes.c_int),
        ("num_ctas", ctypes.c_int),
        ("max_slabs", ctypes.c_int),
        ("ws_floats", ctypes.c_ulonglong),
        ("sem_ints", ctypes.c_int),
        ("cluster", ctypes.c_int),
        ("error", ctypes.c_char * 96),
    ]


MAX_RANKS = 8                   # DG_MAX_RANKS
ERR_GATHER_WAIT = 0x81


class DgGather(ctypes.Structure):
    _fields_ = [
        ("world", ctypes.c_int),
        ("rank", ctypes.c_int),
        ("ldo", ctypes.c_int),
        ("outputs", ctypes.c_void_p * MAX_RANKS),
        ("flags", ctypes.c_void_p * MAX_RANKS),
        ("sync", ctypes.c_void_p),
    ]


class DgGatherLines(ctypes.Structure):
    _fields_ = [
        ("world", ctypes.c_int),
        ("rank", ctypes.c_int),
        ("ldo", ctypes.c_int),
        ("output", ctypes.c_void_p),
        ("lines", ctypes.c_void_p * MAX_RANKS),
        ("sync", ctypes.c_void_p),
        ("q_out", ctypes.c_void_p),
        ("q_scales", ctypes.c_void_p),
    ]


class DgBlockTables(ctypes.Structure):
    _fields_ = [
        ("batch", ctypes.c_int),
        ("page_size", ctypes.c_int),
        ("table_width", ctypes.c_int),
        ("num_tokens", ctypes.c_int),
        ("free_count", ctypes.c_int),
        ("table_stride", ctypes.c_longlong),
        ("context_lens", ctypes.c_void_p),
        ("new_lens", ctypes.c_void_p),
        ("free_pages", ctypes.c_void_p),
        ("cursor_in", ctypes.c_void_p),
        ("block_table", ctypes.c_void_p),
        ("seq_lens", ctypes.c_void_p),
        ("query_start", ctypes.c_void_p),
        ("slots", ctypes.c_void_p),
        ("positions", ctypes.c_void_p),
        ("requests", ctypes.c_void_p),
        ("cursor_out", ctypes.c_void_p),
        ("status", ctypes.c_void_p),
    ]


_Stride2 = ctypes.c_longlong * 2
_Stride3 = ctypes.c_longlong * 3


class DgRotaryArgs(ctypes.Structure):
    _fields_ = [
        ("tokens", ctypes.c_int),
        ("heads", ctypes.c_int),
        ("kv_heads", ctypes.c_int),
        ("head_dim", ctypes.c_int),
        ("rot", ctypes.c_int),
        ("type", ctypes.c_int),
        ("cache_type", ctypes.c_int),
        ("pairing", ctypes.c_int),
        ("inverse", ctypes.c_int),
        ("position_64", ctypes.c_int),
        ("max_position", ctypes.c_int),
        ("page_size", ctypes.c_int),
        ("num_pages", ctypes.c_int),
        ("q", ctypes.c_void_p),
        ("k", ctypes.c_void_p),
        ("v", ctypes.c_void_p),
        ("q_out", ctypes.c_void_p),
        ("k_out", ctypes.c_void_p),
        ("k_cache", ctypes.c_void_p),
        ("v_cache", ctypes.c_void_p),
        ("q_stride", _Stride2),
        ("k_stride", _Stride2),
        ("v_stride", _Stride2),
        ("q_out_stride", _Stride2),
        ("k_out_stride", _Stride2),
        ("k_cache_stride", _Stride3),
        ("v_cache_stride", _Stride3),
        ("positions", ctypes.c_void_p),
        ("position_stride", ctypes.c_longlong),
        ("slots", ctypes.c_void_p),
        ("cos_sin", ctypes.c_void_p),
        ("k_scale", ctypes.c_void_p),
        ("v_scale", ctypes.c_void_p),
        ("status", ctypes.c_void_p),
        ("axis_of", ctypes.c_uint * (MAX_ROT // 32)),
    ]


class DgAttentionArgs(ctypes.Structure):
    _fields_ = [
        ("batch", ctypes.c_int),
        ("heads", ctypes.c_int),
        ("kv_heads", ctypes.c_int),
        ("head_dim", ctypes.c_int),
        ("page_size", ctypes.c_int),
        ("num_pages", ctypes.c_int),
        ("table_width", ctypes.c_int),
        ("type", ctypes.c_int),
        ("cache_type", ctypes.c_int),
        ("window", ctypes.c_int),
        ("scale", ctypes.c_float),
        ("softcap", ctypes.c_float),
        ("q", ctypes.c_void_p),
        ("k_cache", ctypes.c_void_p),
        ("v_cache", ctypes.c_void_p),
        ("q_stride", _Stride2),
        ("k_cache_stride", _Stride3),
        ("v_cache_stride", _Stride3),
        ("block_table", ctypes.c_void_p),
        ("table_stride", ctypes.c_longlong),
        ("seq_lens", ctypes.c_void_p),
        ("k_scale", ctypes.c_void_p),
        ("v_scale", ctypes.c_void_p),
        ("out", ctypes.c_void_p),
        ("out_stride", _Stride2),
        ("lse", ctypes.c_void_p),
        ("q_out", ctypes.c_void_p),
        ("q_scales", ctypes.c_void_p),
        ("workspace", ctypes.c_void_p),
        ("workspace_bytes", ctypes.c_ulonglong),
        ("status", ctypes.c_void_p),
    ]


TensorMap = ctypes.c_uint8 * 128
IpcHandle = ctypes.c_uint8 * 64

_LIB = None


def lib():
    """Load the library (raises if it has not been built)."""
    global _LIB
    if _LIB is not None:
        return _LIB
    if not os.path.exists(LIB_PATH):
        raise RuntimeError(
            f"{LIB_PATH} is missing: build it with `python -m decode_opt_b200.build` "
            "(there is no non-CUDA implementation of this operator)")
    L = ctypes.CDLL(LIB_PATH)
    cfgp = ctypes.POINTER(DgConfig)
    probp = ctypes.POINTER(DgProblem)
    L.dg_abi_version.restype = ctypes.c_int
    L.dg_plan.argtypes = [cfgp, ctypes.c_int, ctypes.c_int, ctypes.c_int, ctypes.POINTER(DgPlanInfo)]
    L.dg_max_active_clusters.argtypes = [cfgp, ctypes.c_int, ctypes.c_int, ctypes.c_int,
                                         ctypes.POINTER(ctypes.c_int)]
    L.dg_make_weight_map.argtypes = [cfgp, ctypes.c_void_p, ctypes.c_int, ctypes.c_int, ctypes.c_void_p]
    L.dg_make_activation_map.argtypes = [cfgp, ctypes.c_void_p, ctypes.c_int, ctypes.c_int, ctypes.c_void_p]
    L.dg_launch_with_maps.argtypes = [cfgp, probp, ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p,
                                      ctypes.c_int]
    L.dg_launch_quantized.argtypes = [cfgp, probp, ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p,
                                      ctypes.c_void_p, ctypes.c_void_p, ctypes.c_int]
    L.dg_launch.argtypes = [cfgp, probp, ctypes.c_void_p]
    L.dg_launch_static_scratch.argtypes = [cfgp, probp, ctypes.c_void_p, ctypes.POINTER(DgPlanInfo)]
    L.dg_prepack_weight.argtypes = [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_int, ctypes.c_int,
                                    ctypes.c_int, ctypes.c_int, ctypes.c_void_p]
    L.dg_padded_n.argtypes = [ctypes.c_int, ctypes.c_int]
    L.dg_packed_weight_bytes.argtypes = [ctypes.c_int, ctypes.c_int, ctypes.c_int]
    L.dg_packed_weight_bytes.restype = ctypes.c_ulonglong
    L.dg_status_string.argtypes = [ctypes.c_int]
    L.dg_status_string.restype = ctypes.c_char_p
    L.dg_flush_l2.argtypes = [ctypes.c_void_p, ctypes.c_ulonglong, ctypes.c_void_p]
    L.dg_probe_bulk_stream.argtypes = [ctypes.c_void_p, ctypes.c_ulonglong, ctypes.c_uint, ctypes.c_int,
                                       ctypes.c_int, ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p]
    L.dg_probe_naive_read.argtypes = [ctypes.c_void_p, ctypes.c_ulonglong, ctypes.c_int, ctypes.c_void_p,
                                      ctypes.c_void_p]
    L.dg_num_sms.restype = ctypes.c_int
    L.dg_launch_gather.argtypes = [cfgp, probp, ctypes.POINTER(DgGather), ctypes.c_void_p, ctypes.c_void_p,
                                   ctypes.c_void_p, ctypes.c_int]
    L.dg_quantize_act.argtypes = [ctypes.c_void_p, ctypes.c_int, ctypes.c_int, ctypes.c_int, ctypes.c_void_p,
                                  ctypes.c_void_p, ctypes.c_void_p, ctypes.c_int]
    L.dg_launch_gather_lines.argtypes = [cfgp, probp, ctypes.POINTER(DgGatherLines), ctypes.c_void_p,
                                         ctypes.c_void_p, ctypes.c_void_p, ctypes.c_int]
    L.dg_host_device_pointer.argtypes = [ctypes.c_void_p, ctypes.POINTER(ctypes.c_void_p)]
    L.dg_copy_from_host.argtypes = [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_ulonglong, ctypes.c_void_p,
                                    ctypes.c_int]
    L.dg_gather_wait.argtypes = [ctypes.POINTER(DgGather), ctypes.c_void_p, ctypes.c_ulonglong, ctypes.c_void_p]
    L.dg_ipc_export.argtypes = [ctypes.c_void_p, ctypes.c_void_p, ctypes.POINTER(ctypes.c_ulonglong)]
    L.dg_ipc_import.argtypes = [ctypes.c_void_p, ctypes.c_ulonglong, ctypes.POINTER(ctypes.c_void_p)]
    L.dg_ipc_release.argtypes = [ctypes.c_void_p]
    L.dg_probe_mma.argtypes = [ctypes.c_int, ctypes.c_int, ctypes.c_int, ctypes.c_int, ctypes.c_int, ctypes.c_int,
                               ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p]
    L.dg_build_block_tables.argtypes = [ctypes.POINTER(DgBlockTables), ctypes.c_void_p, ctypes.c_int]
    L.dg_rotary.argtypes = [ctypes.POINTER(DgRotaryArgs), ctypes.c_void_p, ctypes.c_int]
    L.dg_paged_attention.argtypes = [ctypes.POINTER(DgAttentionArgs), ctypes.c_void_p, ctypes.c_int]
    L.dg_attention_workspace_bytes.restype = ctypes.c_ulonglong
    if L.dg_abi_version() != ABI_VERSION:
        raise RuntimeError(f"{LIB_PATH}: ABI version {L.dg_abi_version()} != {ABI_VERSION}")
    _LIB = L
    return L
