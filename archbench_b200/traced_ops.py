"""The operators of ``ssm_ops`` and ``linear_ops`` registered with the dispatcher (``torch.library``), for callers that trace:
``torch.compile`` and ``torch.export`` see one opaque operator with known output shapes and a known backward instead of a
call they cannot look into, and ``torch.jit.trace`` records it.  Plain calls take the extension module directly, which
costs a few microseconds less.

Each public function here has the signature of its namesake in ``ops``.  It brings its arguments to the operator's own
types with traced torch functions, so that their gradients come back in the callers'; the extension checks the rest when
the operator runs.  Absent outputs are empty tensors inside."""

from __future__ import annotations

from typing import Optional

import torch
from torch import Tensor

from . import ssm_ops


def _ext():
    return ssm_ops._EXT or ssm_ops.extension()


def _filled(ts, like: Tensor):
    return tuple(like.new_empty(0) if t is None else t for t in ts)


def _or_none(grads, inputs):
    """Gradients of optional inputs: nothing for those that were absent."""
    return tuple(None if t is None else g for g, t in zip(grads, inputs))


def _wants_grad(*ts) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts)


def _to(t: Optional[Tensor], dtype: torch.dtype) -> Optional[Tensor]:
    return None if t is None else t.to(dtype)


# ---- causal convolution -----------------------------------------------------------------------


@torch.library.custom_op("archbench_b200::causal_conv", mutates_args=())
def _conv(x: Tensor, weight: Tensor, bias: Optional[Tensor], state: Optional[Tensor], lengths: Optional[Tensor], activation: Optional[str],
          want: bool) -> tuple[Tensor, Tensor]:
    return _filled(_ext().causal_conv(x, weight, bias, activation, state, want, lengths), x)


@_conv.register_fake
def _(x, weight, bias, state, lengths, activation, want):
    return x.new_empty(x.shape), x.new_empty((x.shape[0], x.shape[2], weight.shape[1] - 1) if want else (0,))


@torch.library.custom_op("archbench_b200::causal_conv_bwd", mutates_args=())
def _conv_bwd(x: Tensor, weight: Tensor, bias: Optional[Tensor], state: Optional[Tensor], lengths: Optional[Tensor], activation: Optional[str],
              dy: Optional[Tensor], dlast: Optional[Tensor]) -> tuple[Tensor, Tensor, Tensor, Tensor]:
    return _filled(_ext().causal_conv_backward(x, weight, bias, activation, state, lengths, dy, dlast), x)


@_conv_bwd.register_fake
def _(x, weight, bias, state, lengths, activation, dy, dlast):
    return _filled((None if t is None else t.new_empty(t.shape) for t in (x, weight, bias, state)), x)


def _conv_setup(ctx, inputs, output):
    *tensors, ctx.activation, ctx.want = inputs
    ctx.save_for_backward(*tensors)


def _conv_backward(ctx, dy, dlast):
    tensors = ctx.saved_tensors
    return *_or_none(_conv_bwd(*tensors, ctx.activation, dy, dlast if ctx.want else None), tensors[:4]), None, None, None


_conv.register_autograd(_conv_backward, setup_context=_conv_setup)


def causal_conv(x, weight, bias=None, activation=None, initial_state=None, output_final_state=False, lengths=None):
    if weight.dim() == 3 and weight.shape[1] != 1:
        raise ValueError(f"weight must be (C, W) or (C, 1, W), got {tuple(weight.shape)}")
    w = weight[:, 0] if weight.dim() == 3 else weight
    y, last = _conv(x, w, _to(bias, w.dtype), _to(initial_state, x.dtype), lengths, activation, bool(output_final_state))
    return y, last if output_final_state else None


@torch.library.custom_op("archbench_b200::causal_conv_step", mutates_args=("state",))
def _conv_step(x: Tensor, weight: Tensor, state: Tensor, bias: Optional[Tensor], activation: Optional[str]) -> Tensor:
    return _ext().causal_conv_step(x, weight, state, bias, activation)


@_conv_step.register_fake
def _(x, weight, state, bias, activation):
    return x.new_empty(x.shape)


def causal_conv_step(x, weight, state, bias=None, activation=None):
    return _conv_step(x, weight, state, bias, activation)


# ---- selective scan ---------------------------------------------------------------------------


@torch.library.custom_op("archbench_b200::selective_scan", mutates_args=())
def _scan(x: Tensor, dt: Tensor, A: Tensor, B: Tensor, C: Tensor, D: Optional[Tensor], z: Optional[Tensor], dt_bias: Optional[Tensor],
          h0: Optional[Tensor], lengths: Optional[Tensor], softplus: bool, want: bool, train: bool) -> tuple[Tensor, Tensor, Tensor]:
    return _filled(_ext().selective_scan_forward(x, dt, A, B, C, D, z, dt_bias, softplus, h0, want, lengths, train), A)


@_scan.register_fake
def _(x, dt, A, B, C, D, z, dt_bias, h0, lengths, softplus, want, train):
    b, T, d = x.shape
    N = A.shape[1]
    return x.new_empty(x.shape), A.new_empty((b, d, N) if want else (0,)), A.new_empty((b, (T + 7) // 8, d, N) if train else (0,))


@torch.library.custom_op("archbench_b200::selective_scan_bwd", mutates_args=())
def _scan_bwd(x: Tensor, dt: Tensor, A: Tensor, B: Tensor, C: Tensor, D: Optional[Tensor], z: Optional[Tensor], dt_bias: Optional[Tensor],
              h0: Optional[Tensor], lengths: Optional[Tensor], ckpt: Tensor, softplus: bool, dy: Optional[Tensor], dh: Optional[Tensor]
              ) -> tuple[Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor]:
    return _filled(_ext().selective_scan_backward(x, dt, A, B, C, D, z, dt_bias, softplus, h0, lengths, ckpt, dy, dh), A)


@_scan_bwd.register_fake
def _(x, dt, A, B, C, D, z, dt_bias, h0, lengths, ckpt, softplus, dy, dh):
    return _filled((None if t is None else t.new_empty(t.shape) for t in (x, dt, A, B, C, D, z, dt_bias, h0)), A)


def _scan_setup(ctx, inputs, output):
    *tensors, ctx.softplus, ctx.want, _ = inputs
    ctx.save_for_backward(*tensors, output[2])


def _scan_backward(ctx, dy, dh, _):
    tensors = ctx.saved_tensors
    return *_or_none(_scan_bwd(*tensors, ctx.softplus, dy, dh if ctx.want else None), tensors[:9]), None, None, None, None


_scan.register_autograd(_scan_backward, setup_context=_scan_setup)


def _groups(t: Tensor, x: Tensor) -> Tensor:
    return (t.unsqueeze(-2) if t.dim() == x.dim() else t).to(x.dtype)


def selective_scan(x, dt, A, B, C, D=None, z=None, dt_bias=None, dt_softplus=False, initial_state=None, output_final_state=False,
                   lengths=None):
    f32 = torch.float32
    args = (x, dt.to(x.dtype), A.to(f32), _groups(B, x), _groups(C, x), _to(D, f32), _to(z, x.dtype), _to(dt_bias, f32), _to(initial_state, f32))
    y, h, _ = _scan(*args, lengths, bool(dt_softplus), bool(output_final_state), _wants_grad(*args))
    return y, h if output_final_state else None


@torch.library.custom_op("archbench_b200::selective_scan_step", mutates_args=("state",))
def _scan_step(x: Tensor, dt: Tensor, A: Tensor, B: Tensor, C: Tensor, state: Tensor, D: Optional[Tensor], z: Optional[Tensor],
               dt_bias: Optional[Tensor], softplus: bool) -> Tensor:
    return _ext().selective_scan_step(x, dt, A, B, C, state, D, z, dt_bias, softplus)


@_scan_step.register_fake
def _(x, dt, A, B, C, state, D, z, dt_bias, softplus):
    return x.new_empty(x.shape)


def selective_scan_step(x, dt, A, B, C, state, D=None, z=None, dt_bias=None, dt_softplus=False):
    return _scan_step(x, dt, A, B, C, state, D, z, dt_bias, bool(dt_softplus))


# ---- linear -----------------------------------------------------------------------------------


@torch.library.custom_op("archbench_b200::linear", mutates_args=())
def _linear(x: Tensor, weight: Tensor, bias: Optional[Tensor], residual: Optional[Tensor], activation: Optional[str],
            train: bool) -> tuple[Tensor, Tensor]:
    return _filled(_ext().linear_forward(x, weight, bias, activation, residual, train), x)


@_linear.register_fake
def _(x, weight, bias, residual, activation, train):
    shape = (x.shape[0], weight.shape[0])
    return x.new_empty(shape), x.new_empty(shape, dtype=torch.half) if train and activation is not None else x.new_empty(0)


@torch.library.custom_op("archbench_b200::linear_bwd", mutates_args=())
def _linear_bwd(x: Tensor, weight: Tensor, pre: Optional[Tensor], dy: Tensor, activation: Optional[str],
                needs: int) -> tuple[Tensor, Tensor, Tensor]:
    return _filled(_ext().linear_backward(x, weight, pre, dy, activation, needs), x)


@_linear_bwd.register_fake
def _(x, weight, pre, dy, activation, needs):
    return tuple(x.new_empty(s if needs >> i & 1 else 0) for i, s in enumerate((x.shape, weight.shape, weight.shape[:1])))


def _linear_setup(ctx, inputs, output):
    x, weight, _, _, ctx.activation, _ = inputs
    ctx.save_for_backward(x, weight, None if ctx.activation is None else output[1])


def _linear_backward(ctx, dy, _):
    need = ctx.needs_input_grad
    grads = _linear_bwd(*ctx.saved_tensors, dy, ctx.activation, sum(1 << i for i in range(3) if need[i]))
    return *(g if need[i] else None for i, g in enumerate(grads)), dy if need[3] else None, None, None


_linear.register_autograd(_linear_backward, setup_context=_linear_setup)


def linear(x, weight, bias=None, activation=None, residual=None):
    if x.dim() < 1 or weight.dim() != 2 or weight.shape[1] != x.shape[-1]:
        raise ValueError(f"x must be (..., K) and weight (N, K), got {tuple(x.shape)} and {tuple(weight.shape)}")
    N, K = weight.shape
    if residual is not None and tuple(residual.shape) != (*x.shape[:-1], N):
        raise ValueError(f"residual must be {(*x.shape[:-1], N)}, got {tuple(residual.shape)}")
    rows = lambda t, n: None if t is None else t.reshape(-1, n)  # noqa: E731
    args = (rows(x, K), weight, bias, rows(residual, N))
    y, _ = _linear(*args, activation, _wants_grad(*args))
    return y.reshape(*x.shape[:-1], N)
