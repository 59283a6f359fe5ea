"""Operators of a selective-state-space mixer on the library's CUDA kernels (``include/gdn_b200.h``): the depthwise
causal convolution, the selective scan and their one-token forms.

  causal_conv(x, weight, bias=None, activation=None, initial_state=None, output_final_state=False, lengths=None)
      -> (y, final_state | None)
  causal_conv_step(x, weight, state, bias=None, activation=None) -> y                      (state in place)
  selective_scan(x, dt, A, B, C, D=None, z=None, dt_bias=None, dt_softplus=False, initial_state=None,
                 output_final_state=False, lengths=None) -> (y, final_state | None)
  selective_scan_step(x, dt, A, B, C, state, D=None, z=None, dt_bias=None, dt_softplus=False) -> y  (state in place)

All are reachable as ``archbench_b200.ops.<name>``.  CUDA tensors only, bf16 or fp32 token tensors with any strides;
states and sums are fp32.  Calls that need gradients run the backward kernels through autograd (first order).  Under
``torch.compile`` the calls run eagerly between compiled regions."""

from __future__ import annotations

import ctypes
import functools
import struct
from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from .native import SYMBOLS, _check, _check_cuda, _DT, load_library

ACT = {None: 0, "silu": 1, "gelu": 2}
SCAN_CKPT = 8  # GDN_SCAN_CKPT


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


def _p(t: Optional[torch.Tensor]) -> int:
    return 0 if t is None else t.data_ptr()


def eager(fn):
    """Run ``fn`` between compiled regions under ``torch.compile``; a plain call elsewhere (a bare
    ``torch.compiler.disable`` costs each call 1.5 us)."""
    disabled = torch.compiler.disable(fn)

    @functools.wraps(fn)
    def call(*args, **kwargs):
        return disabled(*args, **kwargs) if torch.compiler.is_compiling() else fn(*args, **kwargs)

    return call


def _layout(block) -> str:
    """The struct codes of a ctypes structure's fields, nested ones in place."""
    codes = {ctypes.c_void_p: "P", ctypes.c_int64: "q", ctypes.c_int32: "i", ctypes.c_uint64: "Q", ctypes.c_float: "f"}
    return "".join(codes[t] if t in codes else _layout(t) for _, t in block._fields_)


class Entry:
    """An entry point taking one argument block and a stream.  The block is packed to the layout of its ctypes mirror:
    filling 30 fields of a ctypes structure takes 3 us, packing them a third of that."""

    def __init__(self, name: str, block, need: Optional[str] = None, ws: int = -2):
        self.name, self.need, self.ws, self.run, self.size = name, need, ws, None, None
        codes = "@" + _layout(block)
        self.pack = struct.Struct(codes).pack
        assert struct.calcsize(codes) == ctypes.sizeof(block), block

    def __call__(self, index: int, *values) -> None:
        """Run on device ``index``'s current stream.  ``values`` are the block's fields; with ``need``, the entry point
        that sizes the workspace, the two from place ``ws`` on are set to one taken from torch's allocator for the call."""
        if self.run is None:
            lib = load_library()
            at = lambda n: ctypes.cast(getattr(lib, n), ctypes.c_void_p).value
            call = ctypes.CFUNCTYPE(ctypes.c_int, ctypes.c_char_p, ctypes.c_void_p)
            self.size = self.need and call(at(self.need))
            self.run = call(at(self.name))
        if torch.cuda.current_device() != index:
            with torch.cuda.device(index):
                return self(index, *values)
        block = self.pack(*values)
        if self.need is not None:
            n = ctypes.c_size_t(0)
            status = self.size(block, ctypes.addressof(n))
            if status:
                _check(status)
            if n.value:
                ws = torch.empty(n.value, dtype=torch.uint8, device=torch.device("cuda", index))
                values = list(values)
                i = self.ws % len(values)
                values[i], values[i + 1] = ws.data_ptr(), n.value
                block = self.pack(*values)
        status = self.run(block, torch._C._cuda_getCurrentRawStream(index))
        if status:
            _check(status)


def _token(t: torch.Tensor, name: str, shape, dtype, index: int) -> torch.Tensor:
    """``t`` checked against a shape and a device, in ``dtype`` with a unit last stride."""
    if t.shape != shape:
        raise ValueError(f"{name} must be {tuple(shape)}, got {tuple(t.shape)}")
    if t.get_device() != index:
        raise ValueError(f"{name} must be on cuda:{index}, got {t.device}")
    if t.dtype is not dtype:
        t = t.to(dtype)
    return t if t.stride(-1) == 1 or shape[-1] == 1 else t.contiguous()


def _dense(t: Optional[torch.Tensor], name: str, shape, dtype, index: int) -> Optional[torch.Tensor]:
    return None if t is None else _token(t, name, shape, dtype, index).contiguous()


def _device_of(x: torch.Tensor, name: str) -> int:
    _check_cuda(x)
    if x.dtype not in _DT:
        raise ValueError(f"{name} must be float32 or bfloat16, got {x.dtype}")
    return x.get_device()


def _lengths(lengths, B: int, index: int) -> Optional[torch.Tensor]:
    if lengths is None:
        return None
    if lengths.is_floating_point() or tuple(lengths.shape) != (B,) or lengths.get_device() != index:
        raise ValueError(f"lengths must be an integer tensor of shape ({B},) on cuda:{index}")
    return lengths.to(torch.int32).contiguous()


def _wants_grad(*ts) -> bool:
    if torch.is_grad_enabled():
        for t in ts:
            if t is not None and t.requires_grad:
                return True
    return False


# ---- causal convolution -----------------------------------------------------------------------


_conv_fwd = Entry("gdn_conv_fwd", ConvArgs)
_conv_step = Entry("gdn_conv_step", ConvArgs)
_conv_bwd = Entry("gdn_conv_bwd", ConvBwdArgs, need="gdn_conv_bwd_workspace_bytes")


def _conv_values(x, weight, bias, state, act, lengths, y=None, state_out=None):
    """The fields of ConvArgs."""
    sx, sy = x.stride(), y.stride() if y is not None else (0, 0)
    if x.dim() == 3:
        B, T, C = x.shape
        tx, ty = sx[1], sy[1]
    else:
        (B, C), T, tx, ty = x.shape, 1, 0, 0
    return (x.data_ptr(), weight.data_ptr(), _p(bias), _p(state), _p(state_out), _p(y), _p(lengths), sx[0], tx, sy[0], ty, B, T, C,
            weight.shape[1], act, _DT[x.dtype], _DT[weight.dtype])


def _conv_forward(x, weight, bias, state, act, want_state, lengths):
    B, T, C = x.shape
    y = torch.empty(B, T, C, device=x.device, dtype=x.dtype)
    out = torch.empty(B, C, weight.shape[1] - 1, device=x.device, dtype=x.dtype) if want_state else None
    _conv_fwd(x.get_device(), *_conv_values(x, weight, bias, state, act, lengths, y, out))
    return y, out


class _Conv(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, state, act, want_state, lengths):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x, weight, bias, state, lengths)
        ctx.act = act
        return _conv_forward(x, weight, bias, state, act, want_state, lengths)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dlast):
        x, weight, bias, state, lengths = ctx.saved_tensors
        B, T, C = x.shape
        if dy is None and dlast is None:
            return (None,) * 7
        if x.numel() == 0:
            dstate = None if state is None else torch.zeros_like(state) if dlast is None else dlast
            return torch.zeros_like(x), torch.zeros_like(weight), None if bias is None else torch.zeros_like(bias), dstate, None, None, None
        dy = torch.zeros_like(x) if dy is None else _token(dy, "dy", x.shape, x.dtype, x.get_device())
        dlast = None if dlast is None else dlast.contiguous()
        dx = torch.empty(B, T, C, device=x.device, dtype=x.dtype)
        dw = torch.empty_like(weight)
        db = None if bias is None else torch.empty_like(bias)
        ds = None if state is None else torch.empty_like(state)
        _conv_bwd(x.get_device(), *_conv_values(x, weight, bias, state, ctx.act, lengths), dy.data_ptr(), dy.stride(0), dy.stride(1),
                  _p(dlast), dx.data_ptr(), _p(ds), dw.data_ptr(), _p(db), 0, 0)
        return dx, dw, db, ds, None, None, None


def _conv_params(weight, bias, C, index):
    if weight.dim() == 3 and weight.shape[1] == 1:
        weight = weight[:, 0]  # nn.Conv1d's (C, 1, W)
    if weight.dim() != 2 or weight.shape[0] != C:
        raise ValueError(f"weight must be ({C}, W) or ({C}, 1, W), got {tuple(weight.shape)}")
    if not 2 <= weight.shape[1] <= 4:
        raise ValueError(f"the convolution kernels serve widths 2 to 4, got {weight.shape[1]}")
    if weight.dtype not in _DT:
        raise ValueError(f"weight must be float32 or bfloat16, got {weight.dtype}")
    weight = _dense(weight, "weight", weight.shape, weight.dtype, index)
    return weight, None if bias is None else _dense(bias, "bias", (C,), weight.dtype, index)


def _act(activation, allowed):
    if activation not in allowed:
        raise ValueError(f"activation must be one of {allowed}, got {activation!r}")
    return ACT[activation]


_CONV_ACTS = (None, "silu")


@eager
def causal_conv(x, weight, bias=None, activation=None, initial_state=None, output_final_state=False, lengths=None):
    """Depthwise causal convolution: y_t = act(bias + sum_w weight[:, w] x_{t-W+1+w}).

    x (B, T, C); weight (C, W) or (C, 1, W), W 2 to 4; bias (C); activation None or "silu"; initial_state (B, C, W - 1),
    the inputs before the first token (zeros if None); lengths (B): tokens of each right-padded row (y is 0 past them).
    Returns (y, final_state or None), final_state the last W - 1 inputs, in x's dtype."""
    index = _device_of(x, "x")
    if x.dim() != 3:
        raise ValueError(f"x must be (B, T, C), got {tuple(x.shape)}")
    B, T, C = x.shape
    act = _act(activation, _CONV_ACTS)
    x = _token(x, "x", x.shape, x.dtype, index)
    weight, bias = _conv_params(weight, bias, C, index)
    state = _dense(initial_state, "initial_state", (B, C, weight.shape[1] - 1), x.dtype, index)
    lengths = _lengths(lengths, B, index)
    if _wants_grad(x, weight, bias, state):
        return _Conv.apply(x, weight, bias, state, act, bool(output_final_state), lengths)
    return _conv_forward(x, weight, bias, state, act, bool(output_final_state), lengths)


@eager
def causal_conv_step(x, weight, state, bias=None, activation=None):
    """One token of ``causal_conv``: x (B, C), state (B, C, W - 1) contiguous, in x's dtype, advanced in place.  No
    autograd."""
    index, dt = _device_of(x, "x"), x.dtype
    if x.dim() != 2:
        raise ValueError(f"x must be (B, C), got {tuple(x.shape)}")
    B, C = x.shape
    act = _act(activation, _CONV_ACTS)
    x = _token(x, "x", x.shape, dt, index)
    weight, bias = _conv_params(weight, bias, C, index)
    want = (B, C, weight.shape[1] - 1)
    if state.shape != want or state.dtype is not dt or not state.is_contiguous() or state.get_device() != index:
        raise ValueError(f"state must be a contiguous {want} {dt} tensor on {x.device}: it is updated in place")
    y = torch.empty(B, C, device=x.device, dtype=dt)
    _conv_step(index, *_conv_values(x, weight, bias, state, act, None, y))
    return y


# ---- selective scan ---------------------------------------------------------------------------


_scan_fwd = Entry("gdn_scan_fwd", ScanArgs, need="gdn_scan_workspace_bytes")
_scan_step = Entry("gdn_scan_step", ScanArgs)
_scan_bwd = Entry("gdn_scan_bwd", ScanBwdArgs, need="gdn_scan_bwd_workspace_bytes", ws=len(ScanArgs._fields_) - 2)


def _scan_values(x, dt, A, Bm, Cm, D, z, bias, h0, lengths, softplus, y=None, h_out=None, ckpt=None):
    """The fields of ScanArgs before the workspace."""
    sx, sdt, sB, sC = x.stride(), dt.stride(), Bm.stride(), Cm.stride()
    sz, sy = z.stride() if z is not None else (0, 0), y.stride() if y is not None else (0, 0)
    if x.dim() == 3:
        B, T, Dm = x.shape
        strides = (sx[0], sx[1], sdt[0], sdt[1], *sB[:3], *sC[:3], sz[0], sz[1], sy[0], sy[1])
    else:
        (B, Dm), T = x.shape, 1
        strides = (sx[0], 0, sdt[0], 0, sB[0], 0, sB[1], sC[0], 0, sC[1], sz[0], 0, sy[0], 0)
    return (x.data_ptr(), dt.data_ptr(), Bm.data_ptr(), Cm.data_ptr(), _p(z), A.data_ptr(), _p(D), _p(bias), _p(h0), _p(lengths), _p(y),
            _p(h_out), _p(ckpt), *strides, B, T, Dm, A.shape[1], Bm.shape[-2], _DT[x.dtype], softplus)


def _scan_forward(x, dt, A, Bm, Cm, D, z, bias, h0, lengths, softplus, want_state, train):
    B, T, Dm = x.shape
    N = A.shape[1]
    y = torch.empty(B, T, Dm, device=x.device, dtype=x.dtype)
    h = torch.empty(B, Dm, N, device=x.device, dtype=torch.float32) if want_state else None
    ckpt = torch.empty(B, (T + SCAN_CKPT - 1) // SCAN_CKPT, Dm, N, device=x.device, dtype=torch.float32) if train else None
    _scan_fwd(x.get_device(), *_scan_values(x, dt, A, Bm, Cm, D, z, bias, h0, lengths, softplus, y, h, ckpt), 0, 0)
    return y, h, ckpt


class _Scan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, dt, A, Bm, Cm, D, z, bias, h0, lengths, softplus, want_state):
        ctx.set_materialize_grads(False)
        y, h, ckpt = _scan_forward(x, dt, A, Bm, Cm, D, z, bias, h0, lengths, softplus, want_state, True)
        ctx.save_for_backward(x, dt, A, Bm, Cm, D, z, bias, h0, lengths, ckpt)
        ctx.softplus = softplus
        return y, h

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dh):
        x, dt, A, Bm, Cm, D, z, bias, h0, lengths, ckpt = ctx.saved_tensors
        if dy is None and dh is None:
            return (None,) * 12
        new = lambda t: None if t is None else torch.empty(t.shape, device=t.device, dtype=t.dtype)  # contiguous
        if x.numel() == 0:
            zero = [None if t is None else torch.zeros_like(t) for t in (x, dt, A, Bm, Cm, D, z, bias)]
            return (*zero, None if h0 is None else torch.zeros_like(h0) if dh is None else dh, None, None, None)
        dy = torch.zeros_like(x) if dy is None else _token(dy, "dy", x.shape, x.dtype, x.get_device())
        dh = None if dh is None else dh.contiguous()
        dx, ddt, dA, dB, dC, dD, dz, db, dh0 = (new(t) for t in (x, dt, A, Bm, Cm, D, z, bias, h0))
        _scan_bwd(x.get_device(), *_scan_values(x, dt, A, Bm, Cm, D, z, bias, h0, lengths, ctx.softplus, ckpt=ckpt), 0, 0, dy.data_ptr(),
                  dy.stride(0), dy.stride(1), _p(dh), dx.data_ptr(), ddt.data_ptr(), dB.data_ptr(), dC.data_ptr(), _p(dz), dA.data_ptr(),
                  _p(dD), _p(db), _p(dh0))
        return dx, ddt, dA, dB, dC, dD, dz, db, dh0, None, None, None


def _scan_inputs(x, dt, A, B, C, D, z, dt_bias):
    """Checked inputs: token tensors in x's dtype with unit last strides, B and C (..., G, N), parameters fp32."""
    index, ty, shape, nd = _device_of(x, "x"), x.dtype, x.shape, x.dim()
    tok, Dm = shape[:-1], shape[-1]
    if A.dim() != 2 or A.shape[0] != Dm:
        raise ValueError(f"A must be ({Dm}, N), got {tuple(A.shape)}")
    N = A.shape[1]
    if not 1 <= N <= 64:
        raise ValueError(f"the scan kernels serve 1 to 64 states per channel, got {N}")
    if B.dim() == nd:
        B = B.unsqueeze(-2)
    if C.dim() == nd:
        C = C.unsqueeze(-2)
    G = B.shape[-2] if B.dim() == nd + 1 else 0
    if G < 1 or Dm % G:
        raise ValueError(f"B must be {(*tok, N)} or {(*tok, 'G', N)} with G a divisor of {Dm}, got {tuple(B.shape)}")
    x = _token(x, "x", shape, ty, index)
    dt = _token(dt, "dt", shape, ty, index)
    states = (*tok, G, N)
    B, C = _token(B, "B", states, ty, index), _token(C, "C", states, ty, index)
    if z is not None:
        z = _token(z, "z", shape, ty, index)
    A = _dense(A, "A", A.shape, torch.float32, index)
    return index, x, dt, A, B, C, _dense(D, "D", (Dm,), torch.float32, index), z, _dense(dt_bias, "dt_bias", (Dm,), torch.float32, index)


@eager
def selective_scan(x, dt, A, B, C, D=None, z=None, dt_bias=None, dt_softplus=False, initial_state=None, output_final_state=False,
                   lengths=None):
    """Selective state space scan over a block of tokens.

        s_t = softplus(dt_t + dt_bias) (or dt_t + dt_bias);  h_t = exp(s_t A) h_{t-1} + s_t x_t B_t
        y_t = (C_t . h_t + D x_t) silu(z_t)

    x, dt, z (B, T, D); A (D, N), usually negative; B, C (B, T, N) or (B, T, G, N), group g serving D / G consecutive
    channels; D, dt_bias (D); initial_state (B, D, N) fp32 (zeros if None); lengths (B): tokens of each right-padded row
    (past them y is 0 and the state stays).  N <= 64.  Returns (y, final_state or None): y in x's dtype, the state fp32.
    Training keeps one state per 8 tokens."""
    if x.dim() != 3:
        raise ValueError(f"x must be (B, T, D), got {tuple(x.shape)}")
    index, x, dt, A, B, C, D, z, dt_bias = _scan_inputs(x, dt, A, B, C, D, z, dt_bias)
    h0 = _dense(initial_state, "initial_state", (x.shape[0], x.shape[2], A.shape[1]), torch.float32, index)
    lengths = _lengths(lengths, x.shape[0], index)
    if _wants_grad(x, dt, A, B, C, D, z, dt_bias, h0):
        return _Scan.apply(x, dt, A, B, C, D, z, dt_bias, h0, lengths, bool(dt_softplus), bool(output_final_state))
    return _scan_forward(x, dt, A, B, C, D, z, dt_bias, h0, lengths, bool(dt_softplus), bool(output_final_state), False)[:2]


@eager
def selective_scan_step(x, dt, A, B, C, state, D=None, z=None, dt_bias=None, dt_softplus=False):
    """One token of ``selective_scan``: x, dt, z (B, D), B, C (B, N) or (B, G, N), state (B, D, N) fp32 contiguous,
    advanced in place.  No autograd."""
    if x.dim() != 2:
        raise ValueError(f"x must be (B, D), got {tuple(x.shape)}")
    index, x, dt, A, B, C, D, z, dt_bias = _scan_inputs(x, dt, A, B, C, D, z, dt_bias)
    want = (x.shape[0], x.shape[1], A.shape[1])
    if state.shape != want or state.dtype is not torch.float32 or not state.is_contiguous() or state.get_device() != index:
        raise ValueError(f"state must be a contiguous {want} float32 tensor on {x.device}: it is updated in place")
    y = torch.empty(want[0], want[1], device=x.device, dtype=x.dtype)
    _scan_step(index, *_scan_values(x, dt, A, B, C, D, z, dt_bias, None, None, bool(dt_softplus), y, state), 0, 0)
    return y
