"""Token counts outside 0 .. T, and of every integer type, mean the nearest count inside."""

import pytest
import torch

from archbench_b200 import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,values", [
    (torch.int64, [3, -1, -(2 ** 40), 2 ** 31, 2 ** 32 + 2, 2 ** 62, 9, 0]),
    (torch.int32, [3, -1, -(2 ** 31), 2 ** 31 - 1, 9, 6, 5, 0]),
    (torch.int16, [3, -1, -(2 ** 15), 2 ** 15 - 1, 9, 6, 5, 0]),
    (torch.uint8, [3, 0, 0, 255, 9, 6, 5, 0]),
])
def test_counts_are_clamped(dtype, values):
    B, T = len(values), 5
    g = torch.Generator("cuda").manual_seed(3)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")
    x, w, A, Bm = rnd(B, T, 8), rnd(8, 4), -torch.ones(8, 4, device="cuda"), rnd(B, T, 4)
    n = torch.tensor(values, dtype=dtype, device="cuda")
    m = torch.tensor([min(max(v, 0), T) for v in values], dtype=torch.int32, device="cuda")
    for f in (lambda n: ops.causal_conv(x, w, activation="silu", output_final_state=True, lengths=n),
              lambda n: ops.selective_scan(x, x, A, Bm, Bm, dt_softplus=True, output_final_state=True, lengths=n)):
        for a, b in zip(f(n), f(m)):
            assert torch.equal(a, b)


def test_convolution_reads_nothing_past_a_rows_tokens():
    g = torch.Generator("cuda").manual_seed(4)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")
    for dtype, C in ((torch.float32, 24), (torch.bfloat16, 24), (torch.bfloat16, 7)):
        n = torch.tensor([0, 1, 17, 40], device="cuda")
        v = dict(x=rnd(4, 40, C).to(dtype), weight=rnd(C, 4).to(dtype), bias=rnd(C).to(dtype), state=rnd(4, C, 3).to(dtype))
        dy, dlast = rnd(4, 40, C).to(dtype), rnd(4, C, 3).to(dtype)
        outs = []
        for fill in (None, float("nan"), float("inf")):
            own, d = {k: t.clone() for k, t in v.items()}, dy.clone()
            if fill is not None:
                for b in range(4):
                    own["x"][b, int(n[b]):] = fill
                    d[b, int(n[b]):] = fill
            own = {k: t.requires_grad_() for k, t in own.items()}
            y, last = ops.causal_conv(own["x"], own["weight"], own["bias"], "silu", own["state"], True, n)
            outs.append([y, last, *torch.autograd.grad([y, last], list(own.values()), [d, dlast])])
        for other in outs[1:]:
            for a, b in zip(outs[0], other):
                assert torch.equal(a, b) and torch.isfinite(a).all()
