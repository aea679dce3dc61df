"""ctypes binding of the C ABI in include/ma_api.h (libmonarch_attn.so).

The library is built in-tree by ``build.py``; loading fails loudly when it is
missing -- there is no CPU or PyTorch fallback for the forward pass.
"""
from __future__ import annotations

import ctypes
import importlib.util
import os
import threading

from . import build

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_NAME = "libmonarch_attn.so"
LIB_PATH = os.path.join(HERE, LIB_NAME)

# ma_dtype_t
DTYPE_F32, DTYPE_F16, DTYPE_BF16, DTYPE_E4M3, DTYPE_I8 = 0, 1, 2, 3, 4
# ma_mask_dtype_t
MASK_NONE, MASK_BOOL, MASK_I32, MASK_I64, MASK_F32, MASK_F16, MASK_BF16 = range(7)
# ma_impl_t
IMPL_AUTO, IMPL_GENERIC, IMPL_TC, IMPL_SMALL = 0, 1, 2, 3
IMPL_NAMES = {IMPL_GENERIC: "generic", IMPL_TC: "tc", IMPL_SMALL: "small"}

MA_OK = 0
MA_ERR_INJECTED = 8
MA_ERR_BAD_PARAMS = 9
MA_ERR_DEVICE = -2
MA_STATUS_WAIT_TIMEOUT = 0x1
MA_STATUS_TMEM_FAIL = 0x2
MA_STATUS_BAD_ITEM = 0x4
MA_STATUS_BAD_PAGE = 0x8
MA_STATUS_BAD_LENGTH = 0x10

EXPORTED = (
    "ma_workspace_bytes",
    "ma_fwd",
    "ma_select_impl",
    "ma_error_string",
    "ma_last_error_detail",
    "ma_read_status",
    "ma_last_launch_count",
    "ma_api_version",
    "ma_bwd_workspace_bytes",
    "ma_bwd",
    "ma_cache_write",
    "ma_cache_read",
    "ma_decode_workspace_bytes",
    "ma_decode",
)

_i64x2 = ctypes.c_int64 * 2
_i64x3 = ctypes.c_int64 * 3
_i64x4 = ctypes.c_int64 * 4


class MaFwdParams(ctypes.Structure):
    """Mirror of ``ma_fwd_params`` (include/ma_api.h)."""

    _fields_ = [
        ("struct_size", ctypes.c_uint32),
        ("q", ctypes.c_void_p),
        ("k", ctypes.c_void_p),
        ("v", ctypes.c_void_p),
        ("out", ctypes.c_void_p),
        ("q_stride", _i64x4),
        ("k_stride", _i64x4),
        ("v_stride", _i64x4),
        ("o_stride", _i64x4),
        ("mask", ctypes.c_void_p),
        ("mask_stride", ctypes.c_int64 * 2),
        ("mask_dtype", ctypes.c_int32),
        ("E", ctypes.c_int32),
        ("H", ctypes.c_int32),
        ("N", ctypes.c_int32),
        ("D", ctypes.c_int32),
        ("Dv", ctypes.c_int32),
        ("block_size", ctypes.c_int32),
        ("num_steps", ctypes.c_int32),
        ("pre_pad", ctypes.c_int32),
        ("dtype", ctypes.c_int32),
        ("out_dtype", ctypes.c_int32),
        ("q_scale", ctypes.c_void_p),
        ("k_scale", ctypes.c_void_p),
        ("v_scale", ctypes.c_void_p),
        ("workspace", ctypes.c_void_p),
        ("workspace_bytes", ctypes.c_size_t),
        ("status", ctypes.c_void_p),
        ("impl", ctypes.c_int32),
        ("v_f32", ctypes.c_int32),
        ("status_host", ctypes.c_void_p),
        ("reserved", ctypes.c_int32 * 4),
    ]

    def __init__(self, **kw):
        super().__init__(**kw)
        self.struct_size = ctypes.sizeof(MaFwdParams)


class MaBwdParams(ctypes.Structure):
    """Mirror of ``ma_bwd_params`` (include/ma_api.h)."""

    _fields_ = [
        ("struct_size", ctypes.c_uint32),
        ("fwd", MaFwdParams),
        ("dout", ctypes.c_void_p),
        ("dout_stride", _i64x4),
        ("dq", ctypes.c_void_p),
        ("dk", ctypes.c_void_p),
        ("dv", ctypes.c_void_p),
        ("dq_stride", _i64x4),
        ("dk_stride", _i64x4),
        ("dv_stride", _i64x4),
        ("workspace", ctypes.c_void_p),
        ("workspace_bytes", ctypes.c_size_t),
        ("reserved", ctypes.c_int32 * 8),
    ]

    def __init__(self, **kw):
        super().__init__(**kw)
        self.struct_size = ctypes.sizeof(MaBwdParams)
        self.fwd.struct_size = ctypes.sizeof(MaFwdParams)


class MaKvCache(ctypes.Structure):
    """Mirror of ``ma_kv_cache`` (include/ma_api.h)."""

    _fields_ = [
        ("struct_size", ctypes.c_uint32),
        ("dtype", ctypes.c_int32),
        ("k_pages", ctypes.c_void_p),
        ("v_pages", ctypes.c_void_p),
        ("k_scale", ctypes.c_void_p),
        ("v_scale", ctypes.c_void_p),
        ("k_stride", _i64x3),
        ("v_stride", _i64x3),
        ("ks_stride", _i64x3),
        ("vs_stride", _i64x3),
        ("page_table", ctypes.c_void_p),
        ("page_table_stride", _i64x2),
        ("E", ctypes.c_int32),
        ("Hk", ctypes.c_int32),
        ("D", ctypes.c_int32),
        ("num_pages", ctypes.c_int32),
        ("page_size", ctypes.c_int32),
        ("max_pages", ctypes.c_int32),
        ("status", ctypes.c_void_p),
        ("status_host", ctypes.c_void_p),
        ("reserved", ctypes.c_int32 * 4),
    ]


    def __init__(self, **kw):
        super().__init__(**kw)
        self.struct_size = ctypes.sizeof(MaKvCache)


class MaCacheWriteParams(ctypes.Structure):
    """Mirror of ``ma_cache_write_params`` (include/ma_api.h)."""

    _fields_ = [
        ("struct_size", ctypes.c_uint32),
        ("dtype", ctypes.c_int32),
        ("cache", MaKvCache),
        ("k", ctypes.c_void_p),
        ("v", ctypes.c_void_p),
        ("k_stride", _i64x4),
        ("v_stride", _i64x4),
        ("start", ctypes.c_void_p),
        ("count", ctypes.c_void_p),
        ("T", ctypes.c_int32),
        ("reserved", ctypes.c_int32 * 5),
    ]

    def __init__(self, **kw):
        super().__init__(**kw)
        self.struct_size = ctypes.sizeof(MaCacheWriteParams)
        self.cache.struct_size = ctypes.sizeof(MaKvCache)


class MaCacheReadParams(ctypes.Structure):
    """Mirror of ``ma_cache_read_params`` (include/ma_api.h)."""

    _fields_ = [
        ("struct_size", ctypes.c_uint32),
        ("dtype", ctypes.c_int32),
        ("cache", MaKvCache),
        ("k", ctypes.c_void_p),
        ("v", ctypes.c_void_p),
        ("k_stride", _i64x4),
        ("v_stride", _i64x4),
        ("lengths", ctypes.c_void_p),
        ("mask", ctypes.c_void_p),
        ("N", ctypes.c_int32),
        ("reserved", ctypes.c_int32 * 5),
    ]

    def __init__(self, **kw):
        super().__init__(**kw)
        self.struct_size = ctypes.sizeof(MaCacheReadParams)
        self.cache.struct_size = ctypes.sizeof(MaKvCache)


class MaDecodeParams(ctypes.Structure):
    """Mirror of ``ma_decode_params`` (include/ma_api.h)."""

    _fields_ = [
        ("struct_size", ctypes.c_uint32),
        ("dtype", ctypes.c_int32),
        ("cache", MaKvCache),
        ("q", ctypes.c_void_p),
        ("out", ctypes.c_void_p),
        ("lse", ctypes.c_void_p),
        ("q_stride", _i64x3),
        ("o_stride", _i64x3),
        ("lengths", ctypes.c_void_p),
        ("mask", ctypes.c_void_p),
        ("mask_stride", _i64x2),
        ("workspace", ctypes.c_void_p),
        ("workspace_bytes", ctypes.c_size_t),
        ("sm_scale", ctypes.c_float),
        ("H", ctypes.c_int32),
        ("mask_dtype", ctypes.c_int32),
        ("mask_len", ctypes.c_int32),
        ("reserved", ctypes.c_int32 * 4),
    ]

    def __init__(self, **kw):
        super().__init__(**kw)
        self.struct_size = ctypes.sizeof(MaDecodeParams)
        self.cache.struct_size = ctypes.sizeof(MaKvCache)


_lib = None
_lock = threading.Lock()


def lib_path() -> str:
    return LIB_PATH


def load() -> ctypes.CDLL:
    """Load libmonarch_attn.so (once); raise if it has not been built."""
    global _lib
    if _lib is not None:
        return _lib
    with _lock:
        if _lib is not None:
            return _lib
        if not os.path.exists(LIB_PATH):
            raise RuntimeError(
                f"{LIB_NAME} is not built (expected at {LIB_PATH}); run "
                "`python -c 'import __graft_entry__ as g; g.build()'` from the repository root")
        lib = ctypes.CDLL(LIB_PATH)
        P = ctypes.POINTER(MaFwdParams)
        lib.ma_workspace_bytes.argtypes = [P]
        lib.ma_workspace_bytes.restype = ctypes.c_size_t
        lib.ma_fwd.argtypes = [P, ctypes.c_void_p]
        lib.ma_fwd.restype = ctypes.c_int
        lib.ma_select_impl.argtypes = [P]
        lib.ma_select_impl.restype = ctypes.c_int
        lib.ma_error_string.argtypes = [ctypes.c_int]
        lib.ma_error_string.restype = ctypes.c_char_p
        lib.ma_last_error_detail.argtypes = []
        lib.ma_last_error_detail.restype = ctypes.c_char_p
        lib.ma_read_status.argtypes = [ctypes.c_void_p, ctypes.c_void_p,
                                       ctypes.POINTER(ctypes.c_uint32)]
        lib.ma_read_status.restype = ctypes.c_int
        lib.ma_last_launch_count.argtypes = []
        lib.ma_last_launch_count.restype = ctypes.c_int
        lib.ma_api_version.argtypes = []
        lib.ma_api_version.restype = ctypes.c_int
        PB = ctypes.POINTER(MaBwdParams)
        lib.ma_bwd_workspace_bytes.argtypes = [PB]
        lib.ma_bwd_workspace_bytes.restype = ctypes.c_size_t
        lib.ma_bwd.argtypes = [PB, ctypes.c_void_p]
        lib.ma_bwd.restype = ctypes.c_int
        for name, cls in (("ma_cache_write", MaCacheWriteParams), ("ma_cache_read", MaCacheReadParams),
                          ("ma_decode", MaDecodeParams)):
            getattr(lib, name).argtypes = [ctypes.POINTER(cls), ctypes.c_void_p]
            getattr(lib, name).restype = ctypes.c_int
        lib.ma_decode_workspace_bytes.argtypes = []
        lib.ma_decode_workspace_bytes.restype = ctypes.c_size_t
        _lib = lib
        return lib


_torch_binding = None


def load_torch_binding():
    """The key-value cache's binding for torch tensors (csrc/ma_torch.cpp),
    given the library's entries (once); raise if it has not been built."""
    global _torch_binding
    if _torch_binding is not None:
        return _torch_binding
    lib = load()
    with _lock:
        if _torch_binding is None:
            path = build.binding_path()
            if not os.path.exists(path):
                raise RuntimeError(
                    "the key-value cache's binding for this Python and torch is not built (expected at "
                    f"{path}); run `python -c 'import __graft_entry__ as g; g.build()'` from the "
                    "repository root")
            spec = importlib.util.spec_from_file_location("_ma_torch", path)
            mod = importlib.util.module_from_spec(spec)
            spec.loader.exec_module(mod)
            address = lambda fn: ctypes.cast(fn, ctypes.c_void_p).value
            mod.init(address(lib.ma_cache_write), address(lib.ma_cache_read), address(lib.ma_decode),
                     lib.ma_decode_workspace_bytes())
            _torch_binding = mod
    return _torch_binding


class MonarchAttentionError(RuntimeError):
    """Raised when the C ABI rejects a call or the device reports a failure."""

    def __init__(self, code: int, message: str):
        super().__init__(message)
        self.code = code


def check(rc: int) -> None:
    if rc != MA_OK:
        lib = load()
        msg = lib.ma_error_string(rc).decode()
        detail = lib.ma_last_error_detail().decode()
        raise MonarchAttentionError(rc, f"monarch attention: {msg} (code {rc})"
                                        + (f": {detail}" if detail else ""))
