"""The matrix product with its epilogue, ``linear(x, weight, bias=None, activation=None, residual=None)``, on the library's
tcgen05 kernel (``include/gdn_b200.h``), forward and backward.  Reachable as ``archbench_b200.ops.linear``."""

from __future__ import annotations

import ctypes

import torch
from torch.autograd.function import once_differentiable

from .native import SYMBOLS, _check_cuda
from .ssm_ops import _P, _SZ, Entry, _act, _p, _wants_grad, eager


class LinearArgs(ctypes.Structure):
    """Mirror of gdn_linear_args (include/gdn_b200.h)."""

    _fields_ = [(n, ctypes.c_void_p) for n in ("x", "weight", "bias", "residual", "y", "pre")] + \
               [(n, ctypes.c_int64) for n in ("sx", "sw", "sr", "sy", "M", "N", "K")] + \
               [("act", ctypes.c_int32), ("reserved", ctypes.c_int32), ("workspace", ctypes.c_void_p), ("workspace_bytes", ctypes.c_uint64)]


class LinearBwdArgs(ctypes.Structure):
    """Mirror of gdn_linear_bwd_args (include/gdn_b200.h)."""

    _fields_ = [(n, ctypes.c_void_p) for n in ("x", "weight", "pre", "dy", "dx", "dweight", "dbias")] + \
               [(n, ctypes.c_int64) for n in ("sx", "sw", "sdy", "M", "N", "K")] + \
               [("act", ctypes.c_int32), ("reserved", ctypes.c_int32), ("workspace", ctypes.c_void_p), ("workspace_bytes", ctypes.c_uint64)]


SYMBOLS.update({
    "gdn_linear_workspace_bytes": ([_P(LinearArgs), _SZ], ctypes.c_int),
    "gdn_linear_fwd": ([_P(LinearArgs), ctypes.c_void_p], ctypes.c_int),
    "gdn_linear_bwd_workspace_bytes": ([_P(LinearBwdArgs), _SZ], ctypes.c_int),
    "gdn_linear_bwd": ([_P(LinearBwdArgs), ctypes.c_void_p], ctypes.c_int),
})


_linear_fwd = Entry("gdn_linear_fwd", LinearArgs, need="gdn_linear_workspace_bytes")
_linear_bwd = Entry("gdn_linear_bwd", LinearBwdArgs, need="gdn_linear_bwd_workspace_bytes")


def _forward(x, weight, bias, residual, act, want_pre):
    M, K = x.shape
    N = weight.shape[0]
    y = torch.empty(M, N, device=x.device, dtype=torch.bfloat16)
    pre = torch.empty(M, N, device=x.device, dtype=torch.bfloat16) if want_pre and act else None
    _linear_fwd(x.get_device(), x.data_ptr(), weight.data_ptr(), _p(bias), _p(residual), y.data_ptr(), _p(pre), x.stride(0),
                weight.stride(0), 0 if residual is None else residual.stride(0), N, M, N, K, act, 0, 0, 0)
    return y, pre


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act):
        y, pre = _forward(x, weight, bias, residual, act, True)
        ctx.save_for_backward(x, weight, bias, pre)
        ctx.act = act
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, bias, pre = ctx.saved_tensors
        (M, K), N = x.shape, weight.shape[0]
        need = ctx.needs_input_grad
        new = lambda want, *s: torch.empty(*s, device=x.device, dtype=x.dtype) if want else None
        if M == 0:
            return x.new_zeros(M, K), torch.zeros_like(weight), None if bias is None else torch.zeros_like(bias), dy, None
        if dy.stride(-1) != 1:
            dy = dy.contiguous()
        dx, dw, db = new(need[0], M, K), new(need[1], N, K), new(bias is not None and need[2], N)
        if dx is not None or dw is not None or db is not None:
            _linear_bwd(x.get_device(), x.data_ptr(), weight.data_ptr(), _p(pre), dy.data_ptr(), _p(dx), _p(dw), _p(db), x.stride(0),
                        weight.stride(0), dy.stride(0), M, N, K, ctx.act, 0, 0, 0)
        return dx, dw, db, dy if need[3] else None, None


def _rows(t: torch.Tensor, name: str, shape, index: int) -> torch.Tensor:
    """A bf16 tensor as rows with a unit last stride."""
    if t.shape != shape:
        raise ValueError(f"{name} must be {tuple(shape)}, got {tuple(t.shape)}")
    if t.dtype is not torch.bfloat16:
        raise ValueError(f"{name} must be bfloat16, got {t.dtype}")
    if t.get_device() != index:
        raise ValueError(f"{name} must be on cuda:{index}, got {t.device}")
    if t.dim() != 2:
        t = t.reshape(-1, shape[-1])
    return t if t.stride(-1) == 1 or shape[-1] == 1 else t.contiguous()


_ACTS = (None, "silu", "gelu")


@eager
def linear(x, weight, bias=None, activation=None, residual=None):
    """y = act(x weight^T + bias) + residual, in one kernel where one tile pass serves it.

    x (..., K), weight (N, K), bias (N), residual (..., N), all bf16 with any strides; activation None, "silu" or "gelu"
    (the exact, erf form).  fp32 accumulation and epilogue, one rounding at the end.  Differentiable in x, weight, bias
    and residual; with an activation, training keeps x weight^T + bias in bf16."""
    _check_cuda(x)
    shape, index = x.shape, x.get_device()
    if len(shape) < 1 or weight.dim() != 2 or weight.shape[1] != shape[-1] or not weight.numel():
        raise ValueError(f"x must be (..., K) and weight (N, K), got {tuple(shape)} and {tuple(weight.shape)}")
    act = _act(activation, _ACTS)
    lead, N = shape[:-1], weight.shape[0]
    rows = _rows(x, "x", shape, index) if lead else _rows(x[None], "x", (1, *shape), index)
    w = _rows(weight, "weight", weight.shape, index)
    if bias is not None:
        if bias.shape != (N,) or bias.dtype is not torch.bfloat16 or bias.get_device() != index:
            raise ValueError(f"bias must be a bfloat16 ({N},) tensor on {x.device}")
        bias = bias.contiguous()
    if residual is not None:
        residual = _rows(residual, "residual", (*lead, N), index) if lead else _rows(residual[None], "residual", (1, N), index)
    if _wants_grad(rows, w, bias, residual):
        y = _Linear.apply(rows, w, bias, residual, act)
    else:
        y = _forward(rows, w, bias, residual, act, False)[0]
    return y if len(lead) == 1 else y.reshape(*lead, N)
