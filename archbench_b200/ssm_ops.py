"""Operators of a selective-state-space mixer on the library's CUDA kernels (``include/gdn_b200.h``): the depthwise
causal convolution, the selective scan and their one-token forms.

  causal_conv(x, weight, bias=None, activation=None, initial_state=None, output_final_state=False, lengths=None)
      -> (y, final_state | None)
  causal_conv_step(x, weight, state, bias=None, activation=None) -> y                      (state in place)
  selective_scan(x, dt, A, B, C, D=None, z=None, dt_bias=None, dt_softplus=False, initial_state=None,
                 output_final_state=False, lengths=None) -> (y, final_state | None)
  selective_scan_step(x, dt, A, B, C, state, D=None, z=None, dt_bias=None, dt_softplus=False) -> y  (state in place)

All are reachable as ``archbench_b200.ops.<name>``.  CUDA tensors only, bf16 or fp32 token tensors with any strides, all of
one call in x's dtype (others are converted to it); the scan's state and all sums are fp32.  Calls that need gradients run the backward kernels through autograd (first order;
forward-mode tangents are refused).  Under
``torch.compile``, ``torch.export`` and ``torch.jit.trace`` they are registered operators (``traced_ops``).

The calls themselves -- checks, allocation, autograd nodes -- are compiled (``csrc/torch_ops.cpp``, the extension module
``_torch_ops``); the ctypes structures here mirror the C ABI's argument blocks for callers that drive it directly."""

from __future__ import annotations

import ctypes
import os

import torch

from .native import _PKG, SYMBOLS


class ConvArgs(ctypes.Structure):
    """Mirror of gdn_conv_args (include/gdn_b200.h)."""

    _fields_ = [(n, ctypes.c_void_p) for n in ("x", "weight", "bias", "state_in", "state_out", "y", "lengths")] + \
               [(n, ctypes.c_int64) for n in ("sx_b", "sx_t", "sy_b", "sy_t", "B", "T", "C")] + \
               [(n, ctypes.c_int32) for n in ("width", "act", "dtype", "w_dtype")]


class ConvBwdArgs(ctypes.Structure):
    """Mirror of gdn_conv_bwd_args (include/gdn_b200.h)."""

    _fields_ = [("fwd", ConvArgs), ("dy", ctypes.c_void_p), ("sdy_b", ctypes.c_int64), ("sdy_t", ctypes.c_int64)] + \
               [(n, ctypes.c_void_p) for n in ("dstate_out", "dx", "dstate_in", "dweight", "dbias", "workspace")] + \
               [("workspace_bytes", ctypes.c_uint64)]


class ScanArgs(ctypes.Structure):
    """Mirror of gdn_scan_args (include/gdn_b200.h)."""

    _fields_ = [(n, ctypes.c_void_p) for n in ("x", "dt", "Bm", "Cm", "z", "A", "Dskip", "dt_bias", "h0", "lengths",
                                                 "y", "h_out", "ckpt")] + \
               [(n, ctypes.c_int64) for n in ("sx_b", "sx_t", "sdt_b", "sdt_t", "sB_b", "sB_t", "sB_g", "sC_b", "sC_t", "sC_g",
                                                "sz_b", "sz_t", "sy_b", "sy_t", "B", "T", "D", "N", "G")] + \
               [("dtype", ctypes.c_int32), ("softplus", ctypes.c_int32), ("workspace", ctypes.c_void_p),
                ("workspace_bytes", ctypes.c_uint64)]


class ScanBwdArgs(ctypes.Structure):
    """Mirror of gdn_scan_bwd_args (include/gdn_b200.h)."""

    _fields_ = [("fwd", ScanArgs), ("dy", ctypes.c_void_p), ("sdy_b", ctypes.c_int64), ("sdy_t", ctypes.c_int64)] + \
               [(n, ctypes.c_void_p) for n in ("dh_out", "dx", "ddt", "dB", "dC", "dz", "dA", "dDskip", "ddt_bias", "dh0")]


_P, _SZ = ctypes.POINTER, ctypes.POINTER(ctypes.c_size_t)
SYMBOLS.update({
    "gdn_conv_fwd": ([_P(ConvArgs), ctypes.c_void_p], ctypes.c_int),
    "gdn_conv_step": ([_P(ConvArgs), ctypes.c_void_p], ctypes.c_int),
    "gdn_conv_bwd_workspace_bytes": ([_P(ConvBwdArgs), _SZ], ctypes.c_int),
    "gdn_conv_bwd": ([_P(ConvBwdArgs), ctypes.c_void_p], ctypes.c_int),
    "gdn_scan_workspace_bytes": ([_P(ScanArgs), _SZ], ctypes.c_int),
    "gdn_scan_fwd": ([_P(ScanArgs), ctypes.c_void_p], ctypes.c_int),
    "gdn_scan_step": ([_P(ScanArgs), ctypes.c_void_p], ctypes.c_int),
    "gdn_scan_bwd_workspace_bytes": ([_P(ScanBwdArgs), _SZ], ctypes.c_int),
    "gdn_scan_bwd": ([_P(ScanBwdArgs), ctypes.c_void_p], ctypes.c_int),
})


_EXT = None


def extension():
    """The compiled operator module (built by ``python -m archbench_b200.build``); raises if absent."""
    global _EXT
    if _EXT is None:
        if not os.path.exists(os.path.join(_PKG, "_torch_ops.so")):
            raise FileNotFoundError("archbench_b200/_torch_ops.so is missing: build it with `python -m archbench_b200.build`")
        from . import _torch_ops

        _EXT = _torch_ops
    return _EXT


# (bound here: looked up per call, and with torch.jit.is_tracing, they cost a small call 0.3 us)
_is_compiling, _is_tracing = torch.compiler.is_compiling, torch._C._is_tracing


def tracing() -> bool:
    """Under ``torch.compile``, ``torch.export`` or ``torch.jit.trace``."""
    return _is_compiling() or _is_tracing()


# The functions below call the extension, or where a call is traced their namesakes among the registered operators.


def causal_conv(x, weight, bias=None, activation=None, initial_state=None, output_final_state=False, lengths=None):
    """Depthwise causal convolution: y_t = act(bias + sum_w weight[:, w] x_{t-W+1+w}).

    x (B, T, C); weight (C, W) or (C, 1, W), W 2 to 4; bias (C); activation None or "silu"; initial_state (B, C, W - 1),
    the inputs before the first token (zeros if None); lengths (B): tokens of each right-padded row (y is 0 past them).
    Returns (y, final_state or None), final_state the last W - 1 inputs, in x's dtype."""
    m = traced_ops if _is_compiling() or _is_tracing() else _EXT or extension()
    return m.causal_conv(x, weight, bias, activation, initial_state, output_final_state, lengths)


def causal_conv_step(x, weight, state, bias=None, activation=None):
    """One token of ``causal_conv``: x (B, C), state (B, C, W - 1) contiguous, in x's dtype, advanced in place.  No
    gradient: a backward through its output raises, and a state that requires one is refused."""
    m = traced_ops if _is_compiling() or _is_tracing() else _EXT or extension()
    return m.causal_conv_step(x, weight, state, bias, activation)


def selective_scan(x, dt, A, B, C, D=None, z=None, dt_bias=None, dt_softplus=False, initial_state=None, output_final_state=False,
                   lengths=None):
    """Selective state space scan over a block of tokens.

        s_t = softplus(dt_t + dt_bias) (or dt_t + dt_bias);  h_t = exp(s_t A) h_{t-1} + s_t x_t B_t
        y_t = (C_t . h_t + D x_t) silu(z_t)

    x, dt, z (B, T, D); A (D, N), usually negative; B, C (B, T, N) or (B, T, G, N), group g serving D / G consecutive
    channels; D, dt_bias (D); initial_state (B, D, N) fp32 (zeros if None); lengths (B): tokens of each right-padded row, int32
    for no conversion (past them y is 0 and the state stays).  N <= 64.  Returns (y, final_state or None): y in x's dtype, the state fp32.
    Training keeps one state per 8 tokens."""
    m = traced_ops if _is_compiling() or _is_tracing() else _EXT or extension()
    return m.selective_scan(x, dt, A, B, C, D, z, dt_bias, dt_softplus, initial_state, output_final_state, lengths)


def selective_scan_step(x, dt, A, B, C, state, D=None, z=None, dt_bias=None, dt_softplus=False):
    """One token of ``selective_scan``: x, dt, z (B, D), B, C (B, N) or (B, G, N), state (B, D, N) fp32 contiguous,
    advanced in place.  No gradient, as for ``causal_conv_step``."""
    m = traced_ops if _is_compiling() or _is_tracing() else _EXT or extension()
    return m.selective_scan_step(x, dt, A, B, C, state, D, z, dt_bias, dt_softplus)


from . import traced_ops  # noqa: E402  (which calls this module's extension)
