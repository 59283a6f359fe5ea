"""The gradient of ops.linear's activation is taken at x weight^T + bias itself, not at its bf16 rounding; and the C entry
points' two ways to keep what it needs."""

import ctypes

import pytest
import torch
import torch.nn.functional as F

import ssm_reference as R
from archbench_b200 import linear_ops as L, ops

pytestmark = pytest.mark.gpu


def slope(p, act):
    p = p.detach().requires_grad_()
    return torch.autograd.grad((F.silu if act == "silu" else F.gelu)(p).sum(), p)[0]


# few rows, tiles, tiles with unaligned rows, a split contraction, pairs of CTAs
@pytest.mark.parametrize("M,N,pad", [(16, 64, 0), (40, 61, 1), (300, 128, 0), (200, 61, 1), (100, 1024, 0), (9600, 2048, 0)])
@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_activation_gradient_at_the_unrounded_product(act, M, N, pad):
    """With the identity as weight dx is dp, rounded once.

    What stands between: the kept slope (2^-11 of itself at most in fp16, 2^-25 below its normal range), its evaluation in
    fp32 (a few 2^-24 of 1; the erf form 1.5e-7 / 2 < 2^-23) and dp's rounding to bf16 (2^-8 of itself).  A product rounded
    to bf16 first would be up to 2^-8 off at 1.5, and the slope there by 2^-9 and more of 1."""
    g = torch.Generator("cuda").manual_seed(M + N)
    x = (3 * torch.randn(M, N, generator=g, device="cuda")).bfloat16()
    b = (0.01 * torch.randn(N, generator=g, device="cuda")).bfloat16()
    dy = torch.randn(M, N, generator=g, device="cuda").bfloat16()
    w = torch.eye(N, device="cuda", dtype=torch.bfloat16)
    if pad:
        big = torch.zeros(M, N + 2 * pad + 1, device="cuda", dtype=torch.bfloat16)
        big[:, pad:pad + N] = x
        x = big[:, pad:pad + N]
    xs = x.detach().requires_grad_()
    got = torch.autograd.grad(ops.linear(xs, w, b, act), xs, dy)[0].double()
    want = dy.double() * slope(x.double() + b.double(), act)
    bound = (2.0 ** -8 + 2.0 ** -11 + 2.0 ** -16) * want.abs() + dy.double().abs() * 2.0 ** -21
    assert ((got - want).abs() <= bound).all(), ((got - want).abs() / bound).max().item()


@pytest.mark.parametrize("keep", [0, 1])
@pytest.mark.parametrize("M", [40, 200])
def test_kept_values_of_the_c_entry(M, keep):
    """`pre` holds x weight^T + bias in bf16 (keep 0) or the activation's slope there in fp16 (keep 1), and the backward
    takes either."""
    N, K = 72, 96
    g = torch.Generator("cuda").manual_seed(M)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda").bfloat16()
    x, w, b, dy = rnd(M, K), (rnd(N, K).float() / K ** 0.5).bfloat16(), rnd(N), rnd(M, N)
    y, pre = torch.empty(M, N, device="cuda", dtype=torch.bfloat16), torch.empty(M, N, device="cuda", dtype=[torch.bfloat16, torch.half][keep])
    lib, s, n = ops.load_library(), torch.cuda.current_stream().cuda_stream, ctypes.c_size_t(0)

    def call(fn, a):
        size = lib.gdn_linear_bwd_workspace_bytes if fn.endswith("bwd") else lib.gdn_linear_workspace_bytes
        assert size(ctypes.byref(a), ctypes.byref(n)) == 0
        ws = torch.empty(max(n.value, 1), device="cuda", dtype=torch.uint8)
        a.workspace, a.workspace_bytes = ws.data_ptr(), n.value
        assert getattr(lib, fn)(ctypes.byref(a), s) == 0
        torch.cuda.synchronize()

    call("gdn_linear_fwd", L.LinearArgs(x=x.data_ptr(), weight=w.data_ptr(), bias=b.data_ptr(), y=y.data_ptr(), pre=pre.data_ptr(), sx=K, sw=K, sy=N,
                                        M=M, N=N, K=K, act=2, keep=keep))
    ref = [t.double().requires_grad_() for t in (x, w, b)]
    p = F.linear(*ref)
    want = slope(p, "gelu") if keep else p.detach()
    half = 2.0 ** -11 if keep else 2.0 ** -8
    assert ((pre.double() - want).abs() <= half * want.abs() + 2.0 ** -18).all()
    dx, dw, db = torch.empty_like(x), torch.empty_like(w), torch.empty_like(b)
    call("gdn_linear_bwd", L.LinearBwdArgs(x=x.data_ptr(), weight=w.data_ptr(), pre=pre.data_ptr(), dy=dy.data_ptr(), dx=dx.data_ptr(),
                                           dweight=dw.data_ptr(), dbias=db.data_ptr(), sx=K, sw=K, sdy=N, M=M, N=N, K=K, act=2, keep=keep))
    for a, e in zip((dx, dw, db), torch.autograd.grad(R.linear(*ref, "gelu"), ref, dy.double())):
        # dp's terms and the result are each rounded to bf16 (2^-9 rms), with keep 0 the product before the slope too
        assert ((a.double() - e).norm() <= 2.0 ** -7 * e.norm()).item()
