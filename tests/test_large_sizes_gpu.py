"""Sizes past a grid's second and third dimension: what the forward takes the backward takes too."""

import pytest
import torch

import ssm_reference as R
from archbench_b200 import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("act", [None, "gelu"])
def test_linear_backward_of_many_rows(act):
    """More than 65,535 groups of 64 rows.  Rows are copies of 1024 different ones, so the weight's gradient is a whole
    multiple of theirs plus the last rows'."""
    M, N, K = 65535 * 64 + 65, 16, 8
    g = torch.Generator("cuda").manual_seed(1)
    few = lambda n: torch.randn(1024, n, generator=g, device="cuda").bfloat16()
    at = torch.arange(M, device="cuda") % 1024
    xf, df = few(K), few(N)
    w = torch.randn(N, K, generator=g, device="cuda").bfloat16()
    b = torch.randn(N, generator=g, device="cuda").bfloat16()
    own = [xf[at].requires_grad_(), w.clone().requires_grad_(), b.clone().requires_grad_()]
    y = ops.linear(*own, act)
    dx, dw, db = torch.autograd.grad(y, own, df[at])
    ref = [t.double().requires_grad_() for t in (xf, w, b)]
    y0 = R.linear(*ref, act)
    count = torch.bincount(at, minlength=1024).double()
    x0, w0, b0 = torch.autograd.grad(y0, ref, df.double() * count[:, None])
    x0 = x0 / count[:, None]
    # y and dx round once (bf16, 2^-8) and dp before its products (2^-8 of 16 terms); the sums over M rows add M roundings
    # of fp32 at most, of which the blocks' partial sums leave the square root, and dp's 1024 different roundings
    assert ((y.double()[:1024] - y0).abs() <= 2.0 ** -8 * y0.abs() + 1e-5).all()
    assert torch.equal(y[-65:], y[at[-65:]]) and torch.equal(dx[-65:], dx[at[-65:]])
    for got, want in ((dx[:1024], x0), (dw, w0), (db, b0)):
        assert ((got.double() - want).norm() <= 2.0 ** -6 * want.norm()).item(), ((got.double() - want).norm() / want.norm()).item()
