"""Forward-mode derivatives: the kernels have none, and a dual tensor is refused instead of losing its tangent."""

import pytest
import torch
import torch.autograd.forward_ad as fwAD

from archbench_b200 import ops

pytestmark = pytest.mark.gpu


def test_dual_tensors_are_refused():
    g = torch.Generator("cuda").manual_seed(1)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")
    x, w, A, B = rnd(2, 5, 8), rnd(8, 4), -torch.ones(8, 4, device="cuda"), rnd(2, 5, 4)
    xb, wb = rnd(3, 16).bfloat16(), rnd(8, 16).bfloat16()
    sc, ss = torch.zeros(2, 8, 3, device="cuda"), torch.zeros(2, 8, 4, device="cuda")
    with fwAD.dual_level():
        dual = lambda t: fwAD.make_dual(t, torch.ones_like(t))
        calls = [lambda: ops.causal_conv(dual(x), w), lambda: ops.causal_conv(x, dual(w)),
                 lambda: ops.causal_conv(x, w, initial_state=dual(sc)), lambda: ops.causal_conv_step(dual(x[:, 0]), w, sc),
                 lambda: ops.selective_scan(dual(x), x, A, B, B), lambda: ops.selective_scan(x, x, dual(A), B, B),
                 lambda: ops.selective_scan(x, x, A, B, B, initial_state=dual(ss)),
                 lambda: ops.selective_scan_step(x[:, 0], x[:, 0], A, dual(B[:, 0]), B[:, 0], ss),
                 lambda: ops.linear(dual(xb), wb), lambda: ops.linear(xb, wb, residual=dual(rnd(3, 8).bfloat16()))]
        for mode in (torch.enable_grad(), torch.no_grad()):
            with mode:
                for f in calls:
                    with pytest.raises(NotImplementedError, match="forward-mode"):
                        f()
        assert ops.linear(xb, wb).shape == (3, 8)  # plain tensors pass inside the level
