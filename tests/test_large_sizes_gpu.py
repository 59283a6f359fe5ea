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


def test_scan_of_many_rows():
    """More rows than a grid's last dimension: forward, gradients, ragged lengths and the one-token form."""
    B, T, D, N = 65535 + 70, 2, 4, 4
    g = torch.Generator("cuda").manual_seed(2)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")
    v = [rnd(B, T, D), rnd(B, T, D), -torch.rand(D, N, generator=g, device="cuda") - 0.1, rnd(B, T, 1, N), rnd(B, T, 1, N), rnd(D), rnd(B, T, D), rnd(D),
         rnd(B, D, N)]
    n = torch.randint(0, T + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
    dy, dh = rnd(B, T, D), rnd(B, D, N)

    def own(ts):
        x, dt, A, Bm, C, Dk, z, bias, h = ts
        return ops.selective_scan(x, dt, A, Bm, C, D=Dk, z=z, dt_bias=bias, dt_softplus=True, initial_state=h, output_final_state=True, lengths=n)

    def ref(ts):
        x, dt, A, Bm, C, Dk, z, bias, h = ts
        return R.scan(x, dt, A, Bm, C, Dk, z, bias, True, h, n)

    a = [t.clone().requires_grad_() for t in v]
    b = [t.double().cpu().requires_grad_() for t in v]
    oa, ob = own(a), ref(b)
    with torch.no_grad():
        for p, q in zip(own(v), oa):
            assert torch.equal(p, q)
    for p, q in zip(oa, ob):
        R.close(p, q, "out", accumulated=128 + N)
    ga, gb = torch.autograd.grad(oa, a, [dy, dh]), torch.autograd.grad(ob, b, [dy.double().cpu(), dh.double().cpu()])
    for i, (p, q) in enumerate(zip(ga, gb)):
        R.close(p, q, str(i), accumulated=256 + (B * T if i in (2, 5, 7) else D if i in (3, 4) else 0))
    h = v[8].clone()
    y = ops.selective_scan_step(v[0][:, 0], v[1][:, 0], v[2], v[3][:, 0], v[4][:, 0], h, D=v[5], z=v[6][:, 0], dt_bias=v[7], dt_softplus=True)
    cut = [t[:, :1] if t.dim() >= 3 and t.shape[1] == T and i != 8 else t for i, t in enumerate(v)]
    c = lambda t: t.double().cpu()
    y0, h0 = R.scan(*(c(t) for t in cut[:5]), c(v[5]), c(cut[6]), c(v[7]), True, c(v[8]))
    R.close(y, y0[:, 0], "step", accumulated=128)
    R.close(h, h0, "step state", accumulated=128)


def test_unserved_sizes_raise_value_errors():
    """Refused before anything is launched or allocated at that size: broadcast views."""
    x = torch.zeros(1, 1, 1, device="cuda")
    A, w = -torch.ones(2 ** 24 + 1, 1, device="cuda"), torch.zeros(2 ** 24 + 1, 2, device="cuda")
    z = x.expand(1, 1, 2 ** 24 + 1)
    with pytest.raises(ValueError):
        ops.selective_scan(z, z, A, x, x)
    with pytest.raises(ValueError):
        ops.causal_conv(z, w)
    with pytest.raises(ValueError):
        ops.selective_scan_step(z[0], z[0], A, x[0], x[0], torch.zeros(1, 2 ** 24 + 1, 1, device="cuda"))


@pytest.mark.parametrize("N", [5, 8])
def test_scan_of_three_grids_of_rows(N):
    """Every launch past the first starts at its own rows: bf16, the plain and the tiled kernels, two groups, odd strides."""
    B, T, D = 2 * 65535 + 70, 1, 4
    g = torch.Generator("cuda").manual_seed(N)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")
    tok = lambda *s: rnd(*s[:-1], s[-1] + 3).bfloat16()[..., 1:1 + s[-1]]
    v = [tok(B, T, D), tok(B, T, D), -torch.rand(D, N, generator=g, device="cuda") - 0.1, tok(B, T, 2, N), tok(B, T, 2, N), rnd(D), tok(B, T, D), rnd(D), rnd(B, D, N)]
    n = torch.randint(0, T + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
    dy, dh = tok(B, T, D), rnd(B, D, N)
    a, b = [t.detach().requires_grad_() for t in v], [t.double().cpu().requires_grad_() for t in v]
    run = lambda f, ts, **kw: f(*ts[:5], ts[5], ts[6], ts[7], True, ts[8], **kw)
    oa = run(ops.selective_scan, a, output_final_state=True, lengths=n)
    ob = run(R.scan, b, lengths=n)
    for p, q in zip(oa, ob):
        R.close(p, q, "out", accumulated=128 + N)
    ga, gb = torch.autograd.grad(oa, a, [dy, dh]), torch.autograd.grad(ob, b, [dy.double().cpu(), dh.double().cpu()])
    for i, (p, q) in enumerate(zip(ga, gb)):
        R.close(p, q, str(i), accumulated=256 + (B * T if i in (2, 5, 7) else D if i in (3, 4) else 0))
    h = v[8].clone()
    y = ops.selective_scan_step(v[0][:, 0], v[1][:, 0], v[2], v[3][:, 0], v[4][:, 0], h, D=v[5], z=v[6][:, 0], dt_bias=v[7], dt_softplus=True)
    y0, h0 = run(R.scan, [t.detach() for t in b])
    R.close(y, y0[:, 0], "step", accumulated=128)
    R.close(h, h0, "step state", accumulated=128)
