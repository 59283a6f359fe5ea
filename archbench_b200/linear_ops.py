"""The matrix product with its epilogue, ``linear(x, weight, bias=None, activation=None, residual=None)``, on the library's
tcgen05 kernel (``include/gdn_b200.h``), forward and backward.  Reachable as ``archbench_b200.ops.linear``."""

from __future__ import annotations

import ctypes

from . import ssm_ops, traced_ops
from .native import SYMBOLS
from .ssm_ops import _P, _SZ, _is_compiling, _is_tracing


class LinearArgs(ctypes.Structure):
    """Mirror of gdn_linear_args (include/gdn_b200.h)."""

    _fields_ = [(n, ctypes.c_void_p) for n in ("x", "weight", "bias", "residual", "y", "pre")] + \
               [(n, ctypes.c_int64) for n in ("sx", "sw", "sr", "sy", "M", "N", "K")] + \
               [("act", ctypes.c_int32), ("keep", ctypes.c_int32), ("workspace", ctypes.c_void_p), ("workspace_bytes", ctypes.c_uint64)]


class LinearBwdArgs(ctypes.Structure):
    """Mirror of gdn_linear_bwd_args (include/gdn_b200.h)."""

    _fields_ = [(n, ctypes.c_void_p) for n in ("x", "weight", "pre", "dy", "dx", "dweight", "dbias")] + \
               [(n, ctypes.c_int64) for n in ("sx", "sw", "sdy", "M", "N", "K")] + \
               [("act", ctypes.c_int32), ("keep", ctypes.c_int32), ("workspace", ctypes.c_void_p), ("workspace_bytes", ctypes.c_uint64)]


SYMBOLS.update({
    "gdn_linear_workspace_bytes": ([_P(LinearArgs), _SZ], ctypes.c_int),
    "gdn_linear_fwd": ([_P(LinearArgs), ctypes.c_void_p], ctypes.c_int),
    "gdn_linear_bwd_workspace_bytes": ([_P(LinearBwdArgs), _SZ], ctypes.c_int),
    "gdn_linear_bwd": ([_P(LinearBwdArgs), ctypes.c_void_p], ctypes.c_int),
})


def linear(x, weight, bias=None, activation=None, residual=None):
    """y = act(x weight^T + bias) + residual, in one kernel where one tile pass serves it.

    x (..., K), weight (N, K), bias (N), residual (..., N), all bf16 with any strides; activation None, "silu" or "gelu"
    (the erf form).  fp32 accumulation and epilogue, one rounding at the end.  Differentiable in x, weight, bias and
    residual; with an activation, training keeps its slope at x weight^T + bias in fp16."""
    m = traced_ops if _is_compiling() or _is_tracing() else ssm_ops._EXT or ssm_ops.extension()
    return m.linear(x, weight, bias, activation, residual)
