"""Host-side native helpers (C++), loaded with ctypes.

``libmsgl_host.so`` is built from ``csrc/host/*.cpp``: the radix-tree key comparison
(the reference has the same helper in python/minisgl/kernel/csrc/src/radix.cpp:19-40), the
page free-list and the CPU expert GEMV. Each function has a NumPy restatement that is used
when the library has not been built and that the unit tests compare against.
"""
from __future__ import annotations

import ctypes
import os
from typing import Optional

import numpy as np

_HERE = os.path.dirname(os.path.abspath(__file__))
_LIB_PATH = os.path.join(_HERE, "libmsgl_host.so")
_lib: Optional[ctypes.CDLL] = None
_tried = False


def host_lib() -> Optional[ctypes.CDLL]:
    global _lib, _tried
    if _tried:
        return _lib
    _tried = True
    if os.path.exists(_LIB_PATH):
        lib = ctypes.CDLL(_LIB_PATH)
        lib.msgl_common_prefix_i32.restype = ctypes.c_int64
        lib.msgl_common_prefix_i32.argtypes = [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_int64]
        if hasattr(lib, "msgl_prompt_plan"):
            lib.msgl_prompt_plan.restype = ctypes.c_int
            lib.msgl_prompt_plan.argtypes = [ctypes.c_void_p] * 2 + [ctypes.c_int64] * 3 + [ctypes.c_void_p, ctypes.c_int64, ctypes.c_void_p]
        _lib = lib
    return _lib


def common_prefix_len_numpy(a: np.ndarray, b: np.ndarray, limit: int) -> int:
    n = min(limit, len(a), len(b))
    if n == 0:
        return 0
    diff = np.flatnonzero(a[:n] != b[:n])
    return int(diff[0]) if diff.size else n


def common_prefix_len(a: np.ndarray, b: np.ndarray, limit: int) -> int:
    """Length of the common prefix of two int32 arrays, capped at ``limit``."""
    lib = host_lib()
    n = min(limit, len(a), len(b))
    if lib is None or n < 64:
        return common_prefix_len_numpy(a, b, n)
    a = np.ascontiguousarray(a[:n])
    b = np.ascontiguousarray(b[:n])
    return int(lib.msgl_common_prefix_i32(a.ctypes.data, b.ctypes.data, n))


def prompt_tables(cu_q: np.ndarray, seq_lens: np.ndarray, window: int, tile: int):
    """``(tables, t_pad, items, rows, longest request)`` as ``ops.cuda.PrefillPlan`` builds them (``cu_q``, ``seq_lens``: contiguous
    int64); ``None`` where the library was not built."""
    lib = host_lib()
    if lib is None or not hasattr(lib, "msgl_prompt_plan"):
        return None
    if seq_lens.ndim != 1 or cu_q.ndim != 1 or cu_q.size < seq_lens.size + 1:
        raise ValueError(f"first rows {cu_q.shape} of requests {seq_lens.shape}")
    out, info = np.empty(2048, dtype=np.int32), np.empty(5, dtype=np.int64)
    for _ in range(2):
        rc = lib.msgl_prompt_plan(cu_q.ctypes.data, seq_lens.ctypes.data, seq_lens.size, window, tile, out.ctypes.data, out.size,
                                  info.ctypes.data)
        if rc < 0:
            raise ValueError("a request has from 0 to as many rows as tokens, the first at 0 or behind it")
        t_pad, items, rows, longest, words = info.tolist()
        if rc:
            return out[:words], t_pad, items, rows, longest
        out = np.empty(words, dtype=np.int32)
