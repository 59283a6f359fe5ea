"""ops.linear on the GPU against a plain 64-bit form: output and gradients over the kernels' paths (few rows, tiles of
each width, split contractions, rows that TMA cannot address)."""

import pytest
import torch

import ssm_reference as R
from archbench_b200 import ops

pytestmark = pytest.mark.gpu

CASES = [  # M, N, K, bias, act, residual, odd rows (views that start off a 16-byte boundary)
    (1, 8, 8, True, None, True, False),
    (1, 1, 1, True, "silu", True, False),
    (7, 48, 96, True, "gelu", False, False),
    (16, 130, 264, False, None, True, False),
    (31, 33, 77, True, "silu", True, False),
    (64, 200, 520, True, "gelu", True, False),
    (50, 72, 64, True, None, True, True),
    (65, 64, 64, False, None, False, False),
    (128, 256, 128, True, None, True, False),
    (129, 257, 65, True, "gelu", True, False),
    (300, 96, 2048, True, "silu", True, False),    # split contraction
    (200, 264, 1000, False, "silu", False, True),
    (1000, 61, 333, True, None, True, False),
    (2500, 1024, 72, True, "gelu", True, False),   # 128-wide tiles
    (5000, 1024, 136, True, None, True, False),    # 256-wide tiles
    (4777, 1032, 200, False, "silu", True, True),
    (2300, 2048, 320, True, "silu", True, False),  # pairs of CTAs on 256 x 256 tiles
    (9500, 2304, 72, False, "gelu", True, False),
]


def close(got, want, scale, what, roundings):
    """|got - want| <= half a bf16 unit of the value and `roundings` of its terms' (2^-9 relative each, rms-sized sums:
    4 sigma) on top of the fp32 sum's own error; `scale` is the size of the sum."""
    g, w = got.detach().double().cpu(), want.detach().double().cpu()
    assert g.shape == w.shape, what
    bound = 2.0 ** -8 * w.abs() + scale * (2.0 ** -18 + 4 * roundings * 2.0 ** -9)
    worst = ((g - w).abs() / bound).max().item()
    assert torch.isfinite(g).all() and worst <= 1.0, f"{what}: {worst:.3g} times the bound"


def off(t, odd):
    if not odd:
        return t
    big = torch.full((t.shape[0], t.shape[1] + 5), float("nan"), device=t.device, dtype=t.dtype)
    big[:, 3:3 + t.shape[1]] = t
    return big[:, 3:3 + t.shape[1]]


@pytest.mark.parametrize("case", CASES)
def test_linear_forward_and_backward(case):
    M, N, K, bias, act, residual, odd = case
    g = torch.Generator("cuda").manual_seed(M + 3 * N + 7 * K)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda").bfloat16()
    v = dict(x=rnd(M, K), weight=(rnd(N, K).float() / K ** 0.5).bfloat16(), bias=rnd(N) if bias else None, residual=rnd(M, N) if residual else None)
    dy = rnd(M, N)
    ref = {k: None if t is None else t.double().requires_grad_() for k, t in v.items()}
    y0 = R.linear(ref["x"], ref["weight"], ref["bias"], act, ref["residual"])
    with torch.no_grad():
        y = ops.linear(off(v["x"], odd), off(v["weight"], odd), v["bias"], act, None if v["residual"] is None else off(v["residual"], odd))
    close(y, y0, 4.0, "y", 0)
    own = {k: None if t is None else off(t, odd and k in ("x", "weight")).detach().requires_grad_() for k, t in v.items()}
    y = ops.linear(own["x"], own["weight"], own["bias"], act, own["residual"])
    close(y, y0, 4.0, "y", 0)
    names = [k for k in own if own[k] is not None]
    got = torch.autograd.grad(y, [own[k] for k in names], off(dy, odd))
    want = torch.autograd.grad(y0, [ref[k] for k in names], dy.double())
    # dp (and with an activation the stored pre-activation) is rounded to bf16 before the products: sums of M (N) terms
    # of rms size dp x (dp W), each off by 2^-9 relative at most
    r = 0 if act is None else 2
    sizes = dict(x=max(1.0, (N / K) ** 0.5), weight=M ** 0.5, bias=M ** 0.5, residual=1.0)
    for k, a, b in zip(names, got, want):
        close(a, b, sizes[k], "d" + k, r if k != "residual" else 0)


@pytest.mark.parametrize("M,N,K,odd", [(2305, 2056, 1100, False), (2200, 2047, 333, True), (9728, 2304, 200, False), (512, 4096, 5000, False)])
def test_linear_large_tiles(M, N, K, odd):
    """Pairs of CTAs, split contractions and ragged edges of both, with no activation between: each value differs from the
    64-bit one by its own rounding, at most 2^-9 of it, and by fp32 sums' errors (5000 terms: 2^-12 of their rms at most),
    so the difference's 2-norm is within 2^-9 + 2^-12."""
    g = torch.Generator("cuda").manual_seed(M + N)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda").bfloat16()
    x, w, b, r, dy = off(rnd(M, K), odd), off(rnd(N, K), odd), rnd(N), off(rnd(M, N), odd), rnd(M, N)
    ref = [t.double().requires_grad_() for t in (x, w, b, r)]
    own = [t.detach().requires_grad_() for t in (x, w, b, r)]
    y0, y = R.linear(ref[0], ref[1], ref[2], None, ref[3]), ops.linear(own[0], own[1], own[2], None, own[3])
    got, want = [y, *torch.autograd.grad(y, own, dy)], [y0, *torch.autograd.grad(y0, ref, dy.double())]
    for n, a, e in zip("y dx dw db dr".split(), got, want):
        rel = ((a.double() - e).norm() / e.norm()).item()
        assert rel <= 2.0 ** -9 + 2.0 ** -12, (n, rel)
    assert ops.device_status() == 0


def test_linear_shapes_and_partial_gradients():
    g = torch.Generator("cuda").manual_seed(0)
    x = torch.randn(2, 3, 40, generator=g, device="cuda").bfloat16()
    w = torch.randn(24, 40, generator=g, device="cuda").bfloat16()
    y = ops.linear(x, w)
    assert y.shape == (2, 3, 24)
    assert torch.equal(ops.linear(x[0, 0], w), y[0, 0])
    assert torch.equal(ops.linear(x.transpose(0, 1), w), y.transpose(0, 1))
    assert ops.linear(x[:0], w).shape == (0, 3, 24)
    wt = w.t().contiguous().t()  # a weight stored the other way round
    assert torch.equal(ops.linear(x, wt), y)
    wg = w.clone().requires_grad_()
    r = torch.randn(2, 3, 24, generator=g, device="cuda").bfloat16().requires_grad_()
    ops.linear(x, wg, residual=r, activation="silu").sum().backward()
    assert wg.grad.shape == w.shape and torch.equal(r.grad, torch.ones_like(r))
    # a broadcast residual: its gradient is summed over the rows it served
    b = torch.zeros(1, 1, 24, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    ops.linear(x, w, residual=b.expand(2, 3, 24)).sum().backward()
    assert torch.equal(b.grad, torch.full_like(b, 6.0))


def test_linear_is_deterministic():
    g = torch.Generator("cuda").manual_seed(2)
    x = torch.randn(3000, 320, generator=g, device="cuda").bfloat16()
    w = torch.randn(96, 320, generator=g, device="cuda").bfloat16()
    outs = []
    for _ in range(2):
        xs, ws = x.clone().requires_grad_(), w.clone().requires_grad_()
        y = ops.linear(xs, ws, activation="gelu")
        outs.append([y, *torch.autograd.grad(y, [xs, ws], torch.ones_like(y))])
    assert all(torch.equal(a, b) for a, b in zip(*outs))
    assert ops.device_status() == 0


def test_linear_keeps_infinities_in_their_rows():
    x = torch.ones(200, 64, device="cuda", dtype=torch.bfloat16)
    w = torch.ones(72, 64, device="cuda", dtype=torch.bfloat16)
    x[5, 3], x[9, 0] = float("inf"), float("nan")
    y = ops.linear(x, w)
    assert torch.isinf(y[5]).all() and torch.isnan(y[9]).all()
    keep = torch.ones(200, dtype=torch.bool)
    keep[5] = keep[9] = False
    assert (y[keep] == 64).all()


def test_linear_refusals():
    x = torch.zeros(4, 16, device="cuda", dtype=torch.bfloat16)
    w = torch.zeros(8, 16, device="cuda", dtype=torch.bfloat16)
    for f in (lambda: ops.linear(x.cpu(), w), lambda: ops.linear(x.float(), w.float()), lambda: ops.linear(x, w.float()),
              lambda: ops.linear(x, w[:, :8]), lambda: ops.linear(x, w[0]), lambda: ops.linear(x, w, activation="relu"),
              lambda: ops.linear(x, w, bias=torch.zeros(7, device="cuda", dtype=torch.bfloat16)),
              lambda: ops.linear(x, w, bias=torch.zeros(8, device="cuda")),
              lambda: ops.linear(x, w, residual=torch.zeros(4, 7, device="cuda", dtype=torch.bfloat16))):
        with pytest.raises(ValueError):
            f()
