"""ctypes binding of the C ABI in include/rsfa.h (librsfa.so).

The library holds the gfx950 kernels; there is no other compute path.  Loading
fails loudly when the library has not been built.
"""
import ctypes
import os
import threading

_LIB_PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "lib", "librsfa.so")

ABI_VERSION = 6

# rsfa_status
OK = 0
E_NULL = -1
E_SHAPE = -2
E_HEADDIM = -3
E_DTYPE = -4
E_TILE = -5
E_ALIGN = -6
E_DEVICE = -7
E_LAUNCH = -8
E_ABI = -9
E_WORKSPACE = -10
E_SCRATCH = -11
E_ROTARY = -12
E_CACHE = -13
E_BUDGET = -14
E_DRAFT = -15
E_CROSS = -16

# rsfa_dtype
DTYPE_F16 = 0
DTYPE_BF16 = 1
DTYPE_F16_V8E5M2 = 2  # q, k, o float16; v float8_e5m2
DTYPE_F32 = 3  # rsfa_rotary only

# flags
FLAG_STATIC_SCHEDULE = 0x1
FLAG_CAUSAL_SPLIT = 0x2
FLAG_EXACT_TILE = 0x4
FLAG_TILE_HINT = 0x8
FLAG_SINGLE_BLOCKS = 0x10

# rsfa_rotary flags
ROTARY_INTERLEAVED = 0x1
ROTARY_INVERSE = 0x2
ROTARY_POS64 = 0x4

# rsfa_attention_fwd_noalloc's fixed workspace
NOALLOC_WORKSPACE_BYTES = 16 << 20

# most drafted tokens of a call
DRAFT_TOKENS = 512

# Every symbol include/rsfa.h declares, with (restype, argtypes).
_I64 = ctypes.c_int64
_I32 = ctypes.c_int32
_PI32 = ctypes.POINTER(ctypes.c_int32)


class FwdArgs(ctypes.Structure):
    """Mirror of struct rsfa_fwd_args."""

    _fields_ = [
        ("struct_size", ctypes.c_uint32),
        ("dtype", ctypes.c_int32),
        ("q", ctypes.c_void_p),
        ("k", ctypes.c_void_p),
        ("v", ctypes.c_void_p),
        ("o", ctypes.c_void_p),
        ("lse", ctypes.c_void_p),
        ("workspace", ctypes.c_void_p),
        ("workspace_bytes", ctypes.c_uint64),
        ("z", ctypes.c_int64),
        ("h", ctypes.c_int64),
        ("n_ctx", ctypes.c_int64),
        ("head_dim", ctypes.c_int64),
        ("q_stride", ctypes.c_int64 * 4),
        ("k_stride", ctypes.c_int64 * 4),
        ("v_stride", ctypes.c_int64 * 4),
        ("o_stride", ctypes.c_int64 * 4),
        ("sm_scale", ctypes.c_float),
        ("causal", ctypes.c_int32),
        ("block_m", ctypes.c_int32),
        ("block_n", ctypes.c_int32),
        ("flags", ctypes.c_uint32),
    ]


class RotaryArgs(ctypes.Structure):
    """Mirror of struct rsfa_rotary_args."""

    _fields_ = [
        ("struct_size", ctypes.c_uint32),
        ("dtype", ctypes.c_int32),
        ("x", ctypes.c_void_p * 2),
        ("y", ctypes.c_void_p * 2),
        ("z", ctypes.c_int64),
        ("n", ctypes.c_int64),
        ("head_dim", ctypes.c_int64),
        ("rotary_dim", ctypes.c_int64),
        ("heads", ctypes.c_int64 * 2),
        ("x_stride", (ctypes.c_int64 * 4) * 2),
        ("y_stride", (ctypes.c_int64 * 4) * 2),
        ("positions", ctypes.c_void_p),
        ("pos_stride", ctypes.c_int64 * 2),
        ("start", ctypes.c_int64),
        ("turns", ctypes.c_void_p),
        ("amplitude", ctypes.c_float),
        ("flags", ctypes.c_uint32),
    ]


class Cache4(ctypes.Structure):
    """Mirror of struct rsfa_cache4."""

    _fields_ = [
        ("k_codes", ctypes.c_void_p),
        ("k_scales", ctypes.c_void_p),
        ("v_codes", ctypes.c_void_p),
        ("v_scales", ctypes.c_void_p),
        ("positions", ctypes.c_void_p),
        ("weights", ctypes.c_void_p),
        ("z", ctypes.c_int64),
        ("h", ctypes.c_int64),
        ("capacity", ctypes.c_int64),
        ("head_dim", ctypes.c_int64),
        ("code_stride", ctypes.c_int64 * 2),
        ("scale_stride", ctypes.c_int64 * 2),
        ("slot_stride", ctypes.c_int64 * 2),
        ("dtype", ctypes.c_int32),
        ("reserved", ctypes.c_int32),
    ]


class Cache4RowsArgs(ctypes.Structure):
    """Mirror of struct rsfa_cache4_rows_args."""

    _fields_ = [
        ("struct_size", ctypes.c_uint32),
        ("reserved", ctypes.c_uint32),
        ("cache", Cache4),
        ("k", ctypes.c_void_p),
        ("v", ctypes.c_void_p),
        ("t", ctypes.c_int64),
        ("k_stride", ctypes.c_int64 * 4),
        ("v_stride", ctypes.c_int64 * 4),
        ("lengths", ctypes.c_void_p),
        ("length", ctypes.c_int64),
        ("slots", ctypes.c_void_p),
        ("counts", ctypes.c_void_p),
        ("pos_start", ctypes.c_void_p),
    ]


class Cache4AttendArgs(ctypes.Structure):
    """Mirror of struct rsfa_cache4_attend_args."""

    _fields_ = [
        ("struct_size", ctypes.c_uint32),
        ("causal", ctypes.c_int32),
        ("cache", Cache4),
        ("q", ctypes.c_void_p),
        ("o", ctypes.c_void_p),
        ("lse", ctypes.c_void_p),
        ("heads", ctypes.c_int64),
        ("t", ctypes.c_int64),
        ("q_stride", ctypes.c_int64 * 4),
        ("o_stride", ctypes.c_int64 * 4),
        ("lengths", ctypes.c_void_p),
        ("length", ctypes.c_int64),
        ("max_length", ctypes.c_int64),
        ("counts", ctypes.c_void_p),
        ("pos_start", ctypes.c_void_p),
        ("sm_scale", ctypes.c_float),
        ("accumulate", ctypes.c_int32),
        ("workspace", ctypes.c_void_p),
        ("workspace_bytes", ctypes.c_uint64),
    ]


class Cache4EvictArgs(ctypes.Structure):
    """Mirror of struct rsfa_cache4_evict_args."""

    _fields_ = [
        ("struct_size", ctypes.c_uint32),
        ("reserved", ctypes.c_uint32),
        ("cache", Cache4),
        ("into", Cache4),
        ("lengths", ctypes.c_void_p),
        ("length", ctypes.c_int64),
        ("n", ctypes.c_int64),
        ("budget", ctypes.c_int64),
        ("recent", ctypes.c_int64),
        ("sinks", ctypes.c_int64),
        ("out", ctypes.c_void_p),
        ("workspace", ctypes.c_void_p),
        ("workspace_bytes", ctypes.c_uint64),
    ]


class CrossArgs(ctypes.Structure):
    """Mirror of struct rsfa_cross_args."""

    _fields_ = [
        ("struct_size", ctypes.c_uint32),
        ("dtype", ctypes.c_int32),
        ("q", ctypes.c_void_p),
        ("k", ctypes.c_void_p),
        ("v", ctypes.c_void_p),
        ("o", ctypes.c_void_p),
        ("lse", ctypes.c_void_p),
        ("z", ctypes.c_int64),
        ("heads", ctypes.c_int64),
        ("key_heads", ctypes.c_int64),
        ("t", ctypes.c_int64),
        ("n", ctypes.c_int64),
        ("head_dim", ctypes.c_int64),
        ("q_stride", ctypes.c_int64 * 4),
        ("k_stride", ctypes.c_int64 * 4),
        ("v_stride", ctypes.c_int64 * 4),
        ("o_stride", ctypes.c_int64 * 4),
        ("lengths", ctypes.c_void_p),
        ("sm_scale", ctypes.c_float),
        ("reserved", ctypes.c_uint32),
        ("workspace", ctypes.c_void_p),
        ("workspace_bytes", ctypes.c_uint64),
    ]


class CrossBwdArgs(ctypes.Structure):
    """Mirror of struct rsfa_cross_bwd_args."""

    _fields_ = [
        ("struct_size", ctypes.c_uint32),
        ("dtype", ctypes.c_int32),
        ("q", ctypes.c_void_p),
        ("k", ctypes.c_void_p),
        ("v", ctypes.c_void_p),
        ("o", ctypes.c_void_p),
        ("lse", ctypes.c_void_p),
        ("grad_o", ctypes.c_void_p),
        ("grad_lse", ctypes.c_void_p),
        ("grad_q", ctypes.c_void_p),
        ("grad_k", ctypes.c_void_p),
        ("grad_v", ctypes.c_void_p),
        ("z", ctypes.c_int64),
        ("heads", ctypes.c_int64),
        ("key_heads", ctypes.c_int64),
        ("t", ctypes.c_int64),
        ("n", ctypes.c_int64),
        ("head_dim", ctypes.c_int64),
        ("q_stride", ctypes.c_int64 * 4),
        ("k_stride", ctypes.c_int64 * 4),
        ("v_stride", ctypes.c_int64 * 4),
        ("o_stride", ctypes.c_int64 * 4),
        ("grad_o_stride", ctypes.c_int64 * 4),
        ("grad_q_stride", ctypes.c_int64 * 4),
        ("grad_k_stride", ctypes.c_int64 * 4),
        ("grad_v_stride", ctypes.c_int64 * 4),
        ("lengths", ctypes.c_void_p),
        ("sm_scale", ctypes.c_float),
        ("reserved", ctypes.c_uint32),
        ("workspace", ctypes.c_void_p),
        ("workspace_bytes", ctypes.c_uint64),
    ]


class DraftTreeArgs(ctypes.Structure):
    """Mirror of struct rsfa_draft_tree_args."""

    _fields_ = [
        ("struct_size", ctypes.c_uint32),
        ("reserved", ctypes.c_uint32),
        ("parents", ctypes.c_void_p),
        ("parents_stride", ctypes.c_int64),
        ("trees", ctypes.c_int64),
        ("t", ctypes.c_int64),
        ("bits", ctypes.c_void_p),
        ("depths", ctypes.c_void_p),
    ]


class Cache4KeepArgs(ctypes.Structure):
    """Mirror of struct rsfa_cache4_keep_args."""

    _fields_ = [
        ("struct_size", ctypes.c_uint32),
        ("reserved", ctypes.c_uint32),
        ("cache", Cache4),
        ("tokens", ctypes.c_void_p),
        ("n", ctypes.c_int64),
        ("lengths", ctypes.c_void_p),
        ("length", ctypes.c_int64),
        ("counts", ctypes.c_void_p),
        ("pos_start", ctypes.c_void_p),
    ]


SIGNATURES = {
    "rsfa_attention_fwd": (ctypes.c_int, [ctypes.POINTER(FwdArgs), ctypes.c_void_p]),
    "rsfa_attention_fwd_noalloc": (ctypes.c_int, [ctypes.POINTER(FwdArgs), ctypes.c_void_p]),
    "rsfa_split_workspace_bytes": (ctypes.c_uint64, [_I64, _I64, _I64, _I64, _I32]),
    "rsfa_v8_workspace_bytes": (ctypes.c_uint64, [_I64, _I64, _I64, _I64]),
    "rsfa_get_tiling": (ctypes.c_int, [_I64, _I64, _I64, _I64, _I32, _I32, _PI32, _PI32]),
    "rsfa_resolve_tiling": (ctypes.c_int, [_I64, _I32, _I32, _I32, _I32, _PI32, _PI32]),
    "rsfa_get_num_compute_cores": (ctypes.c_int, [ctypes.c_int]),
    "rsfa_rotary": (ctypes.c_int, [ctypes.POINTER(RotaryArgs), ctypes.c_void_p]),
    "rsfa_cache4_append": (ctypes.c_int, [ctypes.POINTER(Cache4RowsArgs), ctypes.c_void_p]),
    "rsfa_cache4_read": (ctypes.c_int, [ctypes.POINTER(Cache4RowsArgs), ctypes.c_void_p]),
    "rsfa_cache4_attend": (ctypes.c_int, [ctypes.POINTER(Cache4AttendArgs), ctypes.c_void_p]),
    "rsfa_cache4_attend_workspace_bytes": (ctypes.c_uint64, [ctypes.POINTER(Cache4AttendArgs)]),
    "rsfa_cache4_claim": (ctypes.c_int, [ctypes.POINTER(Cache4EvictArgs), ctypes.c_void_p]),
    "rsfa_cache4_evict": (ctypes.c_int, [ctypes.POINTER(Cache4EvictArgs), ctypes.c_void_p]),
    "rsfa_cache4_evict_workspace_bytes": (ctypes.c_uint64, [ctypes.POINTER(Cache4EvictArgs), _I32]),
    "rsfa_cross_fwd": (ctypes.c_int, [ctypes.POINTER(CrossArgs), ctypes.c_void_p]),
    "rsfa_cross_fwd_workspace_bytes": (ctypes.c_uint64, [ctypes.POINTER(CrossArgs)]),
    "rsfa_cross_bwd": (ctypes.c_int, [ctypes.POINTER(CrossBwdArgs), ctypes.c_void_p]),
    "rsfa_cross_bwd_workspace_bytes": (ctypes.c_uint64, [ctypes.POINTER(CrossBwdArgs)]),
    "rsfa_draft_tree": (ctypes.c_int, [ctypes.POINTER(DraftTreeArgs), ctypes.c_void_p]),
    "rsfa_cache4_attend_tree": (ctypes.c_int, [ctypes.POINTER(Cache4AttendArgs), ctypes.c_void_p, _I64, ctypes.c_void_p]),
    "rsfa_cache4_attend_tree_workspace_bytes": (ctypes.c_uint64, [ctypes.POINTER(Cache4AttendArgs)]),
    "rsfa_cache4_keep": (ctypes.c_int, [ctypes.POINTER(Cache4KeepArgs), ctypes.c_void_p]),
    "rsfa_strerror": (ctypes.c_char_p, [ctypes.c_int]),
    "rsfa_abi_version": (ctypes.c_int, []),
}

_lib = None
_lock = threading.Lock()


def library_path():
    return _LIB_PATH


def lib():
    """The loaded librsfa.so (raises RuntimeError if it is not built)."""
    global _lib
    if _lib is not None:
        return _lib
    with _lock:
        if _lib is None:
            if not os.path.exists(_LIB_PATH):
                raise RuntimeError(
                    f"ascend_rsfa native library not found at {_LIB_PATH}; build it with "
                    "`python ascend-rsfa_amd/build_native.py` (or __graft_entry__.build())")
            handle = ctypes.CDLL(_LIB_PATH)
            for name, (res, args) in SIGNATURES.items():
                fn = getattr(handle, name)
                fn.restype = res
                fn.argtypes = args
            if handle.rsfa_abi_version() != ABI_VERSION:
                raise RuntimeError("librsfa.so ABI version mismatch; rebuild the library")
            _lib = handle
    return _lib


def strerror(status):
    return lib().rsfa_strerror(status).decode()
