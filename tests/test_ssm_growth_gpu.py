"""Decays above 1 (positive A, or steps without softplus below zero) on rows that are split over time: a state of zero
stays zero however much a segment would have grown it."""

import pytest
import torch

import ssm_reference as R
from archbench_b200 import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("N", [4, 5])
def test_zero_states_do_not_overflow(N):
    T, D = 2048, 8
    g = torch.Generator("cuda").manual_seed(N)
    x, dt = torch.zeros(1, T, D, device="cuda"), torch.full((1, T, D), 4.0, device="cuda")
    x[:, -3:] = torch.randn(1, 3, D, generator=g, device="cuda")  # growth of exp(12) over what follows
    A = torch.ones(D, N, device="cuda")
    Bm, C = torch.randn(1, T, 1, N, generator=g, device="cuda"), torch.randn(1, T, 1, N, generator=g, device="cuda")
    dy = torch.zeros(1, T, D, device="cuda")
    dy[:, :3] = torch.randn(1, 3, D, generator=g, device="cuda")  # gradients that only early tokens make
    own, ref = [t.clone().requires_grad_() for t in (x, dt, A, Bm, C)], [t.double().cpu().requires_grad_() for t in (x, dt, A, Bm, C)]
    y, h = ops.selective_scan(*own, output_final_state=True)
    y0, h0 = R.scan(*ref)
    R.close(y, y0, "y", accumulated=128 + N)
    R.close(h, h0, "state", accumulated=128)
    for a, b, n in zip(torch.autograd.grad(y, own, dy), torch.autograd.grad(y0, ref, dy.double().cpu()), ("x", "dt", "A", "B", "C")):
        R.close(a, b, "d" + n, accumulated=256 + T)
