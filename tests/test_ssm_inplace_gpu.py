"""The one-token operators advance their state in place: autograd sees that write, so a backward that had kept the old
state refuses instead of reading the new one."""

import pytest
import torch

from archbench_b200 import ops

pytestmark = pytest.mark.gpu


def rnd(g, *s):
    return torch.randn(*s, generator=g, device="cuda")


def test_convolution_backward_refuses_an_overwritten_state():
    g = torch.Generator("cuda").manual_seed(1)
    x, w, s = rnd(g, 2, 5, 8), rnd(g, 8, 4).requires_grad_(), rnd(g, 2, 8, 3)
    y, _ = ops.causal_conv(x, w, activation="silu", initial_state=s)
    before = s._version
    ops.causal_conv_step(x[:, 0], w.detach(), s)
    assert s._version > before
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_scan_backward_refuses_an_overwritten_state():
    g = torch.Generator("cuda").manual_seed(2)
    x, A, B, s = rnd(g, 2, 5, 8), -torch.ones(8, 4, device="cuda").requires_grad_(), rnd(g, 2, 5, 4), rnd(g, 2, 8, 4)
    y, _ = ops.selective_scan(x, x, A, B, B, dt_softplus=True, initial_state=s)
    before = s._version
    ops.selective_scan_step(x[:, 0], x[:, 0], A.detach(), B[:, 0], B[:, 0], s, dt_softplus=True)
    assert s._version > before
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_states_of_inference_mode_still_step():
    g = torch.Generator("cuda").manual_seed(3)
    x, w, A, B = rnd(g, 2, 8), rnd(g, 8, 4), -torch.ones(8, 4, device="cuda"), rnd(g, 2, 4)
    with torch.inference_mode():
        sc, ss = torch.zeros(2, 8, 3, device="cuda"), torch.zeros(2, 8, 4, device="cuda")
        ops.causal_conv_step(x, w, sc)
        ops.selective_scan_step(x, x, A, B, B, ss, dt_softplus=True)
    ops.causal_conv_step(x, w, sc)
    ops.selective_scan_step(x, x, A, B, B, ss, dt_softplus=True)
    assert torch.equal(sc[..., 2], x) and ss.abs().sum() > 0
