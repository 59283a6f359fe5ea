"""ops.linear without rows: the residual is checked and keeps its place in the graph."""

import pytest
import torch

from archbench_b200 import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shape", [(0,), (0, 3), (2, 0)])
def test_residual_of_no_rows(shape):
    x, w = torch.zeros(*shape, 16, device="cuda", dtype=torch.bfloat16), torch.ones(8, 16, device="cuda", dtype=torch.bfloat16)
    r = torch.zeros(*shape, 8, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    for act in (None, "silu"):
        y = ops.linear(x, w, None, act, r)
        assert y.shape == r.shape and y.requires_grad
        (g,) = torch.autograd.grad(y, r, torch.zeros_like(y))
        assert g.shape == r.shape
    wg, xg = w.clone().requires_grad_(), x.clone().requires_grad_()
    gw, gx = torch.autograd.grad(ops.linear(xg, wg, None, "gelu", r), (wg, xg), torch.zeros_like(r))
    assert torch.equal(gw, torch.zeros_like(w)) and gx.shape == x.shape
    with pytest.raises(ValueError):
        ops.linear(x, w, residual=torch.zeros(*shape, 7, device="cuda", dtype=torch.bfloat16))
