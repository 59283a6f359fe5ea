"""``SelectiveSSM`` -- a selective-state-space mixer on this package's operators, and ``FusedMLP`` beside it.

    x, z = in_proj(u);  x = silu(conv(x));  r, B, C = x_proj(x);  dt = dt_proj(r)
    h_t = exp(s_t A) h_{t-1} + s_t x_t B_t,  s = softplus(dt + bias);  y = (C . h + D x) silu(z);  out_proj(y) [+ residual]

It is the diagonal counterpart of the gated-DeltaNet mixers (registry name ``ssm``, ``LM(arch="ssm")``): the same call
``forward(x)`` and the same ``GDNCache`` for prompts and single tokens, so ``decode.greedy_decode`` and its CUDA graph
serve it.  Four projections run as ``ops.linear`` (the output projection with the block's residual in its epilogue), the
convolution as ``ops.causal_conv`` and the recurrence as ``ops.selective_scan``, each with its backward; one token without
gradients takes ``ops.causal_conv_step`` and ``ops.selective_scan_step``, which advance the cache in place.  bf16 activations use the
package's matrix product; fp32 ones take ``torch.nn.functional.linear``."""

from __future__ import annotations

import math
from typing import Optional

import torch
import torch.nn as nn
import torch.nn.functional as F

from . import ops
from .layers import GDNCache, _put, _training
from .ssm_ops import tracing


def _linear(x, weight, bias=None, activation=None, residual=None):
    """``ops.linear`` in bf16; the same formula from torch's functions for fp32 activations.  A residual of another type
    than the activations (the fp32 stream of a model under autocast) is added outside the product and keeps its type."""
    weight, bias = weight.to(x.dtype), None if bias is None else bias.to(x.dtype)
    if x.dtype == torch.bfloat16:
        fused = residual is None or residual.dtype == x.dtype
        y = ops.linear(x, weight, bias, activation, residual if fused else None)
        return y if fused else y + residual
    y = F.linear(x, weight, bias)
    y = y if activation is None else F.silu(y) if activation == "silu" else F.gelu(y)
    return y if residual is None else y + residual


def _plain(m: nn.Module, kind: type = nn.Linear) -> bool:
    """True for an ``nn.Linear`` (``nn.Conv1d``) that is its weight and bias and nothing else.  A replacement (an adapter, a
    quantised layer), a parametrised layer or one with hooks runs through its own call."""
    return type(m) is kind and not (m._forward_hooks or m._forward_pre_hooks or m._backward_hooks or m._backward_pre_hooks
                                or "forward" in m.__dict__)


def _project(m: nn.Module, x, activation=None, residual=None):
    """activation(m(x)) + residual, in one product where ``m`` is a plain ``nn.Linear``."""
    if _plain(m):
        return _linear(x, m.weight, m.bias, activation, residual)
    y = m(x)
    y = y if activation is None else F.silu(y) if activation == "silu" else F.gelu(y)
    return y if residual is None else y + residual


def _activations(x: torch.Tensor) -> torch.Tensor:
    """``x`` in the dtype of an enclosing autocast region."""
    return x.to(torch.get_autocast_dtype("cuda")) if torch.is_autocast_enabled("cuda") else x


class SelectiveSSM(nn.Module):
    """Selective-state-space mixer.  ``expand`` times the model width of channels, ``state_size`` states each (at most
    64), ``conv_size`` taps (2 to 4), step sizes through a projection of rank ``dt_rank`` (d_model / 16 rounded up by
    default) that start log-uniform in [dt_min, dt_max]."""

    fuses_residual = True  # forward takes the block's residual and adds it, in the output projection if the types agree

    def __init__(self, d_model: int, layer_idx: int = 0, expand: float = 2.0, state_size: int = 16, conv_size: int = 4,
                 dt_rank: Optional[int] = None, dt_min: float = 1e-3, dt_max: float = 1e-1, bias: bool = False, conv_bias: bool = True):
        super().__init__()
        if not 1 <= state_size <= 64:
            raise ValueError(f"state_size must be 1 to 64, got {state_size}")
        if not 2 <= conv_size <= 4:
            raise ValueError(f"conv_size must be 2 to 4, got {conv_size}")
        self.d_model, self.layer_idx, self.state_size, self.conv_size = d_model, layer_idx, state_size, conv_size
        self.d_inner = int(expand * d_model)
        self.dt_rank = math.ceil(d_model / 16) if dt_rank is None else dt_rank
        Di, R, N = self.d_inner, self.dt_rank, state_size
        self.in_proj = nn.Linear(d_model, 2 * Di, bias=bias)
        self.conv1d = nn.Conv1d(Di, Di, conv_size, groups=Di, padding=conv_size - 1, bias=conv_bias)
        self.x_proj = nn.Linear(Di, R + 2 * N, bias=False)
        self.dt_proj = nn.Linear(R, Di, bias=True)
        self.A_log = nn.Parameter(torch.log(torch.arange(1, N + 1, dtype=torch.float32)).repeat(Di, 1))
        self.D = nn.Parameter(torch.ones(Di))
        self.out_proj = nn.Linear(Di, d_model, bias=bias)
        with torch.no_grad():
            step = torch.exp(torch.rand(Di) * (math.log(dt_max) - math.log(dt_min)) + math.log(dt_min))
            self.dt_proj.bias.copy_(step + torch.log(-torch.expm1(-step)))  # softplus of it is the step

    bound_cache: Optional[GDNCache] = None  # used when called without a cache (decode.bind_caches)

    def _parameters_f32(self, train: bool):
        """A, D and the step bias (None where ``dt_proj`` adds it itself) in fp32; kept between calls while the parameters are
        unchanged, except in training and where the call is traced."""
        bias = self.dt_proj.bias if _plain(self.dt_proj) else None
        if train or tracing():
            return -torch.exp(self.A_log.float()), self.D.float(), None if bias is None else bias.float()
        return (ops._cached(self.A_log, "neg_exp", lambda t: -torch.exp(t.float())), ops._cached(self.D, "f32", lambda t: t.float()),
                None if bias is None else ops._cached(bias, "f32", lambda t: t.float()))

    def _convolve(self, u: torch.Tensor, cache: Optional[GDNCache], one: bool) -> torch.Tensor:
        """silu(conv1d(u)) from the cache's last inputs, which move on; ``one``: in place."""
        c, state = self.conv1d, None if cache is None else cache.conv.get("x")
        if _plain(c, nn.Conv1d):
            weight, bias = c.weight.to(u.dtype), None if c.bias is None else c.bias.to(u.dtype)
            if one:
                return ops.causal_conv_step(u[:, 0], weight, state, bias, "silu")[:, None]
            y, last = ops.causal_conv(u, weight, bias, "silu", state, cache is not None)
        else:  # it pads conv_size - 1 inputs on both sides, as the nn.Conv1d does
            W, T = self.conv_size, u.shape[1]
            past = u.new_zeros(u.shape[0], u.shape[2], W - 1) if state is None else state.to(u.dtype)
            inputs = torch.cat([past, u.transpose(1, 2)], -1)
            y = F.silu(c(inputs)[..., W - 1:W - 1 + T]).transpose(1, 2)
            last = inputs[..., T:].contiguous()
        if cache is not None:
            _put(cache, "x", last)
        return y

    def forward(self, x: torch.Tensor, cache: Optional[GDNCache] = None, residual: Optional[torch.Tensor] = None) -> torch.Tensor:
        if cache is None:
            cache = self.bound_cache
        x = _activations(x)
        T, R, N, train = x.shape[1], self.dt_rank, self.state_size, _training(x, self)
        A, D, dt_bias = self._parameters_f32(train)
        # the one-token forms have no gradient; where one is wanted one token takes the prompt's
        one = cache is not None and cache.state is not None and T == 1 and (
            cache.static or not (train or torch.is_grad_enabled() and cache.state.requires_grad))
        u, z = _project(self.in_proj, x).chunk(2, -1)
        u = self._convolve(u, cache, one)
        r, B, C = _project(self.x_proj, u).split([R, N, N], -1)
        # a plain projection's bias is added to the step sizes inside the scan, in fp32
        dt = _linear(r, self.dt_proj.weight) if dt_bias is not None else self.dt_proj(r)
        if one:
            y = ops.selective_scan_step(u[:, 0], dt[:, 0], A, B[:, 0], C[:, 0], cache.state, D=D, z=z[:, 0], dt_bias=dt_bias,
                                        dt_softplus=True)[:, None]
        else:
            y, state = ops.selective_scan(u, dt, A, B, C, D=D, z=z, dt_bias=dt_bias, dt_softplus=True,
                                          initial_state=None if cache is None else cache.state, output_final_state=cache is not None)
            if cache is not None:
                cache.state = state
        if cache is not None:
            cache.seen += T
        return _project(self.out_proj, y, residual=residual)


class FusedMLP(nn.Module):
    """down(act(up(x))) [+ residual] with biases, each product with its epilogue; ``activation`` "silu" or "gelu"."""

    fuses_residual = True

    def __init__(self, d_model: int, ratio: float, activation: str):
        super().__init__()
        if activation not in ("silu", "gelu"):
            raise ValueError(f"activation must be 'silu' or 'gelu', got {activation!r}")
        hidden = (int(ratio * d_model) + 63) // 64 * 64
        self.activation = activation
        self.up = nn.Linear(d_model, hidden)
        self.down = nn.Linear(hidden, d_model)

    def forward(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None) -> torch.Tensor:
        x = _activations(x)
        return _project(self.down, _project(self.up, x, self.activation), residual=residual)
