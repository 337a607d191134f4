"""ctypes binding of ``librpa_bounded.so`` (the C ABI declared in ``include/rpa_bounded.h``).

Built in-tree next to this file (``tpu_cake_amd.build``); ``RPA_BOUNDED_LIB`` overrides the path.
There is no fallback: if the library is missing every entry point raises.
"""

from __future__ import annotations

import ctypes
import os
import pathlib
import threading

from ._lib import RPA_KV_BF16, RPA_KV_FP8_E4M3, RpaError  # noqa: F401
from ._sparse_lib import ERR_FREE, ERR_LEN, ERR_PAGE, ERR_SLOT, _i32, _struct, _sz, _vp  # noqa: F401

LIB_PATH = pathlib.Path(__file__).with_name("librpa_bounded.so")
ABI_VERSION = 1

_i64, _float = ctypes.c_int64, ctypes.c_float

RpaRotateShape = _struct("RpaRotateShape", *((n, _i32) for n in (
    "num_tokens", "num_q_heads", "num_kv_heads", "head_dim", "rotated", "interleaved", "max_num_seqs", "weight_bytes")),
    *((n, _i64) for n in ("q_token_stride", "q_head_stride", "k_token_stride", "k_head_stride", "q_out_token_stride",
                          "q_out_head_stride", "k_out_token_stride", "k_out_head_stride", "q_weight_stride", "k_weight_stride")))
RpaWeighShape = _struct("RpaWeighShape", *((n, _i32) for n in (
    "num_tokens", "num_q_heads", "num_kv_heads", "head_dim", "total_pages", "page_size", "max_num_seqs", "pages_per_seq",
    "kv_dtype", "reserved")), ("q_token_stride", _i64), ("q_head_stride", _i64))
RpaWeighOptions = _struct("RpaWeighOptions", *((n, _float) for n in ("sm_scale", "soft_cap", "k_scale", "v_scale", "decay")))
RpaChooseShape = _struct("RpaChooseShape", *((n, _i32) for n in (
    "max_num_seqs", "pages_per_seq", "num_kv_heads", "total_pages", "page_size", "budget", "limit", "sinks", "recent",
    "max_moves")))
RpaMoveShape = _struct("RpaMoveShape", *((n, _i32) for n in (
    "num_lists", "max_moves", "num_kv_heads", "head_dim", "total_pages", "page_size", "kv_dtype")))

# name -> (result, argument types): every symbol include/rpa_bounded.h declares
_SIGNATURES = {
    "rpa_bounded_abi_version": (ctypes.c_int, []),
    "rpa_bounded_last_error": (ctypes.c_char_p, []),
    "rpa_bounded_read_error_word": (ctypes.c_int, [ctypes.POINTER(_i32), _i32, _vp]),
    "rpa_rotate_heads": (ctypes.c_int, [ctypes.POINTER(RpaRotateShape)] + [_float] * 2 + [_vp] * 12),
    "rpa_weigh_workspace_size": (_sz, [ctypes.POINTER(RpaWeighShape)]),
    "rpa_weighed_attention": (ctypes.c_int, [ctypes.POINTER(RpaWeighShape), ctypes.POINTER(RpaWeighOptions)] + [_vp] * 12
                              + [_sz, _vp]),
    "rpa_choose_workspace_size": (_sz, [ctypes.POINTER(RpaChooseShape)]),
    "rpa_choose_moves": (ctypes.c_int, [ctypes.POINTER(RpaChooseShape)] + [_vp] * 8 + [_sz, _vp]),
    "rpa_move_rows": (ctypes.c_int, [ctypes.POINTER(RpaMoveShape)] + [_vp] * 6),
}
EXPORTED_SYMBOLS = tuple(_SIGNATURES)

_lock = threading.Lock()
_lib: ctypes.CDLL | None = None


def library_path() -> pathlib.Path:
    return pathlib.Path(os.environ.get("RPA_BOUNDED_LIB", str(LIB_PATH)))


def load() -> ctypes.CDLL:
    """Load ``librpa_bounded.so`` once; raise if it is missing or has the wrong ABI."""
    global _lib
    if _lib is not None:
        return _lib
    with _lock:
        if _lib is not None:
            return _lib
        path = library_path()
        if not path.exists():
            raise RuntimeError(
                f"librpa_bounded.so not found at {path}; build it with `python -m tpu_cake_amd.build` "
                "(there is no CPU fallback)")
        lib = ctypes.CDLL(str(path))
        for name, (result, args) in _SIGNATURES.items():
            fn = getattr(lib, name)
            fn.restype, fn.argtypes = result, args
        version = lib.rpa_bounded_abi_version()
        if version != ABI_VERSION:
            raise RuntimeError(f"{path}: ABI version {version}, expected {ABI_VERSION}")
        _lib = lib
        return lib


def check(rc: int) -> None:
    if rc != 0:
        raise RpaError(rc, load().rpa_bounded_last_error().decode(errors="replace"))


def read_error_word(device=None, *, clear: bool = False) -> int:
    """The error word of ``device`` (default: the current one): bits ``ERR_PAGE``, ``ERR_SLOT``,
    ``ERR_LEN``, ``ERR_FREE`` of all calls since they were last cleared.  Waits for the current stream;
    ``clear`` takes back the bits it returns."""
    import torch

    word = _i32(0)
    with torch.cuda.device(device):
        stream = torch.cuda.current_stream().cuda_stream
        check(load().rpa_bounded_read_error_word(ctypes.byref(word), int(clear), stream))
    return int(word.value)
