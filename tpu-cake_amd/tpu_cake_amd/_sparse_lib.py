"""ctypes binding of ``librpa_sparse.so`` (the C ABI declared in ``include/rpa_sparse.h``).

Built in-tree next to this file (``tpu_cake_amd.build``); ``RPA_SPARSE_LIB`` overrides the path.
There is no fallback: if the library is missing every entry point raises.
"""

from __future__ import annotations

import ctypes
import os
import pathlib
import threading

from ._lib import RPA_KV_BF16, RPA_KV_FP8_E4M3, RpaError  # noqa: F401

LIB_PATH = pathlib.Path(__file__).with_name("librpa_sparse.so")
ABI_VERSION = 1

# bits of the error word
ERR_PAGE, ERR_SLOT, ERR_LEN, ERR_FREE = 1, 2, 4, 8

_vp, _sz, _i32 = ctypes.c_void_p, ctypes.c_size_t, ctypes.c_int32


def _struct(name: str, *fields: tuple) -> type:
    return type(name, (ctypes.Structure,), {"_fields_": list(fields)})


RpaPagingShape = _struct("RpaPagingShape", *((n, _i32) for n in (
    "num_requests", "pages_per_seq", "page_size", "free_capacity", "max_tokens")))
RpaAppendShape = _struct("RpaAppendShape", *((n, _i32) for n in (
    "num_tokens", "num_kv_heads", "head_dim", "total_pages", "page_size", "kv_dtype")), *((n, ctypes.c_int64) for n in (
        "k_token_stride", "k_head_stride", "v_token_stride", "v_head_stride")))
RpaSparseShape = _struct("RpaSparseShape", *((n, _i32) for n in (
    "num_tokens", "num_q_heads", "num_kv_heads", "head_dim", "total_pages", "page_size", "max_num_seqs", "pages_per_seq",
    "kv_dtype", "num_pages")), ("q_token_stride", ctypes.c_int64), ("q_head_stride", ctypes.c_int64))
RpaSparseOptions = _struct("RpaSparseOptions", *((n, ctypes.c_float) for n in ("sm_scale", "soft_cap", "k_scale", "v_scale")))

# name -> (result, argument types): every symbol include/rpa_sparse.h declares
_SIGNATURES = {
    "rpa_sparse_abi_version": (ctypes.c_int, []),
    "rpa_sparse_last_error": (ctypes.c_char_p, []),
    "rpa_sparse_read_error_word": (ctypes.c_int, [ctypes.POINTER(_i32), _i32, _vp]),
    "rpa_assign_pages": (ctypes.c_int, [ctypes.POINTER(RpaPagingShape)] + [_vp] * 12),
    "rpa_release_pages": (ctypes.c_int, [ctypes.POINTER(RpaPagingShape)] + [_vp] * 8),
    "rpa_append_kv": (ctypes.c_int, [ctypes.POINTER(RpaAppendShape)] + [_vp] * 5 + [ctypes.c_float] * 2 + [_vp] * 3),
    "rpa_select_workspace_size": (_sz, [ctypes.POINTER(RpaSparseShape)]),
    "rpa_select_pages": (ctypes.c_int, [ctypes.POINTER(RpaSparseShape), _i32, _i32] + [_vp] * 9 + [_sz, _vp]),
    "rpa_sparse_workspace_size": (_sz, [ctypes.POINTER(RpaSparseShape)]),
    "rpa_sparse_paged_attention": (ctypes.c_int, [ctypes.POINTER(RpaSparseShape), ctypes.POINTER(RpaSparseOptions)]
                                   + [_vp] * 10 + [_sz, _vp]),
}
EXPORTED_SYMBOLS = tuple(_SIGNATURES)

_lock = threading.Lock()
_lib: ctypes.CDLL | None = None


def library_path() -> pathlib.Path:
    return pathlib.Path(os.environ.get("RPA_SPARSE_LIB", str(LIB_PATH)))


def load() -> ctypes.CDLL:
    """Load ``librpa_sparse.so`` once; raise if it is missing or has the wrong ABI."""
    global _lib
    if _lib is not None:
        return _lib
    with _lock:
        if _lib is not None:
            return _lib
        path = library_path()
        if not path.exists():
            raise RuntimeError(
                f"librpa_sparse.so not found at {path}; build it with `python -m tpu_cake_amd.build` "
                "(there is no CPU fallback)")
        lib = ctypes.CDLL(str(path))
        for name, (result, args) in _SIGNATURES.items():
            fn = getattr(lib, name)
            fn.restype, fn.argtypes = result, args
        version = lib.rpa_sparse_abi_version()
        if version != ABI_VERSION:
            raise RuntimeError(f"{path}: ABI version {version}, expected {ABI_VERSION}")
        _lib = lib
        return lib


def check(rc: int) -> None:
    if rc != 0:
        raise RpaError(rc, load().rpa_sparse_last_error().decode(errors="replace"))


def read_error_word(device=None, *, clear: bool = False) -> int:
    """The error word of ``device`` (default: the current one): bits ``ERR_PAGE``, ``ERR_SLOT``,
    ``ERR_LEN``, ``ERR_FREE`` of all calls since they were last cleared.  Waits for the current stream;
    ``clear`` takes back the bits it returns."""
    import torch

    word = _i32(0)
    with torch.cuda.device(device):
        stream = torch.cuda.current_stream().cuda_stream
        check(load().rpa_sparse_read_error_word(ctypes.byref(word), int(clear), stream))
    return int(word.value)
