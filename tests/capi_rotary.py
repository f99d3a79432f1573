"""ctypes view of the rotation part of the C ABI (include/vlak_b200.h)."""
from __future__ import annotations

import ctypes

from kernels import _native


class RotaryTensor(ctypes.Structure):
    _fields_ = [("x", ctypes.c_void_p), ("grad", ctypes.c_void_p), ("y", ctypes.c_void_p),
                ("weight", ctypes.c_void_p), ("grad_weight", ctypes.c_void_p),
                ("H", ctypes.c_int64), ("x_stride", ctypes.c_int64 * 3),
                ("grad_stride", ctypes.c_int64 * 3)]


class RotaryArgs(ctypes.Structure):
    _fields_ = [("t", RotaryTensor * 2), ("positions", ctypes.c_void_p),
                ("inv_freq", ctypes.c_void_p), ("B", ctypes.c_int64), ("M", ctypes.c_int64),
                ("D", ctypes.c_int64), ("rotary_dim", ctypes.c_int64),
                ("pos_stride", ctypes.c_int64 * 2), ("amplitude", ctypes.c_double),
                ("eps", ctypes.c_double), ("n_tensors", ctypes.c_int), ("dtype", ctypes.c_int),
                ("pos_dtype", ctypes.c_int), ("weight_dtype", ctypes.c_int),
                ("interleaved", ctypes.c_int), ("inverse", ctypes.c_int)]


def lib():
    L = _native.capi()
    p, s, n = ctypes.POINTER(RotaryArgs), ctypes.c_void_p, ctypes.c_int64
    L.vlak_rotary.argtypes = [p, s]
    L.vlak_qk_norm_rotary_fwd.argtypes = [p, s]
    L.vlak_qk_norm_rotary_workspace_size.argtypes = [p, ctypes.POINTER(n)]
    L.vlak_qk_norm_rotary_bwd.argtypes = [p, ctypes.c_void_p, n, s]
    return L
