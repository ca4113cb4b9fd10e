"""ctypes binding of ``lib/libs4d_decoder.so`` (the C ABI declared in ``include/s4d_decoder.h``).

The library is loaded on first use.  If it is missing, every operator of it raises instead of
falling back to another implementation.
"""
from __future__ import annotations

import ctypes as C
import os
import threading

import torch

from . import _lib as L

# The in-tree build; S4D_DECODER_LIB may point at another build of the same ABI.
LIB_PATH = os.environ.get("S4D_DECODER_LIB") or os.path.join(os.path.dirname(os.path.abspath(__file__)), "lib",
                                                             "libs4d_decoder.so")

S4D_DTYPE_F16 = 2
DTYPES = {torch.float32: L.S4D_DTYPE_F32, torch.bfloat16: L.S4D_DTYPE_BF16, torch.float16: S4D_DTYPE_F16}

_i64, _int, _p, _sz, _f = C.c_int64, C.c_int, C.c_void_p, C.c_size_t, C.c_float



class AttentionArgs(C.Structure):
    """``s4d_attention_args``.  ``keep`` (not part of the struct) holds the tensors it points to."""

    _fields_ = [(n, _i64) for n in ("batch", "queries", "keys", "heads", "kv_heads", "dim", "pos_dim")] + [
        ("q", _p), ("k", _p), ("v", _p), ("q_stride", _i64 * 3), ("k_stride", _i64 * 3), ("v_stride", _i64 * 3),
        ("out", _p), ("lse", _p), ("slopes", _p), ("slope_stride", _i64 * 3), ("q_pos", _p), ("k_pos", _p),
        ("q_segment", _p), ("k_segment", _p), ("k_len", _p), ("workspace", _p), ("workspace_bytes", _sz),
        ("error_flag", _p), ("scale", _f), ("softcap", _f), ("dtype", C.c_int32),
        ("dslopes_per_row", C.c_int32), ("dout", _p), ("dout_stride", _i64 * 3), ("dq", _p), ("dk", _p), ("dv", _p),
        ("dslopes", _p)]


# name -> (restype, argtypes); one entry per function of include/s4d_decoder.h
SIGNATURES = {
    "s4d_decoder_abi_version": (_int, []),
    "s4d_decoder_last_error": (C.c_char_p, []),
    "s4d_attention_forward_workspace_bytes": (_sz, [C.POINTER(AttentionArgs)]),
    "s4d_attention_forward": (_int, [C.POINTER(AttentionArgs), _p]),
    "s4d_attention_backward_workspace_bytes": (_sz, [C.POINTER(AttentionArgs)]),
    "s4d_attention_backward": (_int, [C.POINTER(AttentionArgs), _p]),
    "s4d_norm_forward": (_int, [_p, _i64, _int, _p, _p, _int, _p, _i64, _p, _p, _i64, _i64, _f, _p]),
    "s4d_norm_backward_workspace_bytes": (_sz, [_i64, _i64]),
    "s4d_norm_backward": (_int, [_p, _i64, _p, _i64, _int, _p, _int, _p, _p, _p, _i64, _p, _p, _i64, _i64, _p, _sz,
                                 _p]),
}

# Version of include/s4d_decoder.h these bindings are written for (s4d_decoder_abi_version()).
ABI_VERSION = 1

_lib = None
_lock = threading.Lock()


def lib():
    global _lib
    if _lib is None:
        with _lock:
            if _lib is None:
                if not os.path.exists(LIB_PATH):
                    raise RuntimeError(
                        f"CUDA library {LIB_PATH} is not built; run `python __graft_entry__.py build` "
                        "(or python sparse4d-tt_b200/build.py).  There is no CPU fallback.")
                handle = C.CDLL(LIB_PATH)
                for name, (res, args) in SIGNATURES.items():
                    fn = getattr(handle, name)
                    fn.restype = res
                    fn.argtypes = args
                version = handle.s4d_decoder_abi_version()
                if version != ABI_VERSION:
                    raise RuntimeError(f"{LIB_PATH} has C ABI version {version}, these bindings expect "
                                       f"{ABI_VERSION}; rebuild it (python sparse4d-tt_b200/build.py)")
                _lib = handle
    return _lib


def check(fn: str, status: int) -> None:
    if status != L.S4D_OK:
        msg = lib().s4d_decoder_last_error().decode()
        if status in (L.S4D_ERR_INVALID_ARG, L.S4D_ERR_UNSUPPORTED_SHAPE):
            raise ValueError(f"{fn}: {L.status_string(status)}: {msg}")
        raise L.S4DError(fn, status, msg)


class on_device:
    """``with on_device(dev):`` makes ``dev`` the current device for the launches inside (they go to
    its current stream); costs nothing when it already is."""

    __slots__ = ("guard",)

    def __init__(self, dev: torch.device):
        self.guard = None if dev.index == torch.cuda.current_device() else torch.cuda.device(dev)

    def __enter__(self):
        if self.guard is not None:
            self.guard.__enter__()

    def __exit__(self, *exc):
        if self.guard is not None:
            self.guard.__exit__(*exc)
        return False
