"""ctypes binding of ``lib/libs4d_decoder.so`` (the C ABI declared in ``include/s4d_decoder.h``), and
the module that takes the calls which need nothing but launches (``csrc/decoder_calls.cpp``).

The library is loaded on first use.  If it is missing, every operator of it raises instead of
falling back to another implementation.
"""
from __future__ import annotations

import ctypes as C
import importlib.machinery
import importlib.util
import os
import struct
import threading

import torch

from . import _lib as L
from .build import calls_path

# The in-tree build; S4D_DECODER_LIB may point at another build of the same ABI.
LIB_PATH = os.environ.get("S4D_DECODER_LIB") or os.path.join(os.path.dirname(os.path.abspath(__file__)), "lib",
                                                             "libs4d_decoder.so")

S4D_DTYPE_F16 = 2
DTYPES = {torch.float32: L.S4D_DTYPE_F32, torch.bfloat16: L.S4D_DTYPE_BF16, torch.float16: S4D_DTYPE_F16}

_i64, _int, _p, _sz, _f = C.c_int64, C.c_int, C.c_void_p, C.c_size_t, C.c_float



# s4d_attention_args as one format of the struct module: packing all fields at once costs a few microseconds
# less a call than setting them one by one.  Pointers are 0 for NULL.
ATTENTION_ARGS = struct.Struct(
    "@7q"   # batch, queries, keys, heads, kv_heads, dim, pos_dim
    "3P"    # q, k, v
    "9q"    # strides of q, k, v
    "3P3q"  # out, lse, slopes and their strides
    "5P"    # q_pos, k_pos, q_segment, k_segment, k_len
    "PNP"   # workspace, workspace_bytes, error_flag
    "2f2i"  # scale, softcap, dtype, dslopes_per_row
    "P3q"   # dout and its strides
    "4P")   # dq, dk, dv, dslopes


# name -> (restype, argtypes); one entry per function of include/s4d_decoder.h
SIGNATURES = {
    "s4d_decoder_abi_version": (_int, []),
    "s4d_decoder_last_error": (C.c_char_p, []),
    "s4d_decoder_set_wait_limit_ns": (C.c_uint64, [C.c_uint64]),
    "s4d_attention_forward_workspace_bytes": (_sz, [C.c_char_p]),
    "s4d_attention_forward": (_int, [C.c_char_p, _p]),
    "s4d_attention_backward_workspace_bytes": (_sz, [C.c_char_p]),
    "s4d_attention_backward": (_int, [C.c_char_p, _p]),
    "s4d_norm_forward": (_int, [_p, _i64, _int, _p, _p, _int, _p, _i64, _p, _p, _i64, _i64, _f, _p]),
    "s4d_norm_backward_workspace_bytes": (_sz, [_i64, _i64]),
    "s4d_norm_backward": (_int, [_p, _i64, _p, _i64, _int, _p, _int, _p, _p, _p, _i64, _p, _p, _i64, _i64, _p, _sz,
                                 _p]),
}

# Version of include/s4d_decoder.h these bindings are written for (s4d_decoder_abi_version()).
ABI_VERSION = 2

_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
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


_calls = None


def calls():
    """The module of csrc/decoder_calls.cpp, over the functions of ``lib()``.  Each of its calls answers None
    for what is not its to take."""
    global _calls
    if _calls is None:
        handle = lib()
        with _lock:
            if _calls is None:
                path = calls_path()
                if not os.path.exists(path):
                    raise RuntimeError(f"{path} is not built (it goes with this Python and torch); run "
                                       "`python __graft_entry__.py build` (or python sparse4d-tt_b200/build.py).")
                loader = importlib.machinery.ExtensionFileLoader("s4d_decoder_calls", path)
                module = importlib.util.module_from_spec(importlib.util.spec_from_loader(loader.name, loader))
                loader.exec_module(module)
                module.init(*(C.cast(getattr(handle, n), C.c_void_p).value for n in (
                    "s4d_norm_forward", "s4d_norm_backward_workspace_bytes", "s4d_norm_backward",
                    "s4d_attention_forward_workspace_bytes", "s4d_attention_forward",
                    "s4d_attention_backward_workspace_bytes", "s4d_attention_backward")))
                _calls = module
    return _calls


def check(fn: str, status: int) -> None:
    if status != L.S4D_OK:
        msg = lib().s4d_decoder_last_error().decode()
        if status in (L.S4D_ERR_INVALID_ARG, L.S4D_ERR_UNSUPPORTED_SHAPE):
            raise ValueError(f"{fn}: {L.status_string(status)}: {msg}")
        raise L.S4DError(fn, status, msg)


class on_device:
    """``with on_device(index):`` makes CUDA device ``index`` the current one for the launches inside (they
    go to its current stream); costs next to nothing when it already is."""

    __slots__ = ("guard",)

    def __init__(self, index: int):
        self.guard = None if index == torch._C._cuda_getDevice() else torch.cuda.device(index)

    def __enter__(self):
        if self.guard is not None:
            self.guard.__enter__()

    def __exit__(self, *exc):
        if self.guard is not None:
            self.guard.__exit__(*exc)
        return False


def in_memory(t: torch.Tensor | None) -> torch.Tensor | None:
    """``t`` such that its memory holds its values: a copy of a view that stands for the negative of its memory (the
    imaginary part of a conjugate)."""
    return t.resolve_neg() if t is not None and t.is_neg() else t


def same_device(name: str, first: torch.Tensor, *others) -> int:
    """The CUDA device index of ``first``, which every other tensor (None: left out) has to share."""
    index = first.get_device()
    if index < 0:
        raise ValueError(f"{name}: every tensor must be on a CUDA device (got {first.device}); no CPU path exists")
    for t in others:
        if t is not None and t.get_device() != index:
            if t.get_device() < 0:
                raise ValueError(f"{name}: every tensor must be on a CUDA device (got {t.device}); no CPU path exists")
            raise ValueError(f"{name}: tensors on different devices (cuda:{index} and {t.device})")
    return index


def overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether the memory from one tensor's first to its last element meets the other's."""
    if a.numel() == 0 or b.numel() == 0:
        return False
    lo, hi = [], []
    for t in (a, b):
        lo.append(t.data_ptr())
        hi.append(t.data_ptr() + t.element_size() * (1 + sum((n - 1) * st for n, st in zip(t.shape, t.stride()))))
    return lo[0] < hi[1] and lo[1] < hi[0]


def stream_ptr(index: int) -> int:
    """torch's current-stream handle of a device index."""
    if _raw_stream is not None:
        return _raw_stream(index)
    return torch.cuda.current_stream(index).cuda_stream
