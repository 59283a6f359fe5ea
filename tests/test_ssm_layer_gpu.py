"""The selective-state-space mixer, the fused MLP and a decoder of them: against the same formulas in 64 bits, in training
and in cached decoding (eager, CUDA graph, torch.compile)."""

import copy

import pytest
import torch
import torch.nn.functional as F

import ssm_reference as R
from archbench_b200.decode import bind_caches, greedy_decode
from archbench_b200.layers import GDNCache
from archbench_b200.lm import LM
from archbench_b200.ssm_layer import FusedMLP, SelectiveSSM

pytestmark = pytest.mark.gpu


def reference_layer(m: SelectiveSSM, x, residual=None):
    """The mixer's formula with the module's (64-bit) parameters."""
    u, z = F.linear(x, m.in_proj.weight, m.in_proj.bias).chunk(2, -1)
    u, _ = R.conv(u, m.conv1d.weight[:, 0], m.conv1d.bias, silu=True)
    r, B, C = F.linear(u, m.x_proj.weight).split([m.dt_rank, m.state_size, m.state_size], -1)
    y, _ = R.scan(u, F.linear(r, m.dt_proj.weight), -torch.exp(m.A_log), B[:, :, None], C[:, :, None], m.D, z, m.dt_proj.bias, True)
    y = F.linear(y, m.out_proj.weight, m.out_proj.bias)
    return y if residual is None else y + residual


def rel(a, b):
    a, b = a.detach().double().cpu(), b.detach().double().cpu()
    return ((a - b).norm() / b.norm()).item()


def make(dtype, **kw):
    torch.manual_seed(3)
    m = SelectiveSSM(64, **kw)
    for p in m.parameters():
        if p.dim() > 1 and p is not m.A_log:
            torch.nn.init.normal_(p, std=0.3 / p[0].numel() ** 0.5 * 3)
    return m.cuda().to(dtype)


# Relative error in the 2-norm.  fp32: torch's fp32 projections (2^-24 per product, sums of 128) and the kernels', well
# under 1e-5.  bf16: about ten roundings of 2^-9 / sqrt(3) = 1.1e-3 along the chain of a gradient, squared sums 4e-3;
# the decays multiply a step size's rounding by s A h / h < 1.  Bound: 1e-2.
@pytest.mark.parametrize("dtype,tol", [(torch.float32, 1e-5), (torch.bfloat16, 1e-2)])
@pytest.mark.parametrize("kw", [dict(), dict(state_size=24, conv_size=3, bias=True), dict(expand=1.5, dt_rank=5, conv_bias=False)])
def test_layer_forward_and_gradients(dtype, tol, kw):
    m = make(dtype, **kw)
    x = torch.randn(2, 37, 64, device="cuda", generator=torch.Generator("cuda").manual_seed(1)).to(dtype)
    res = torch.randn(2, 37, 64, device="cuda", generator=torch.Generator("cuda").manual_seed(2)).to(dtype)
    dy = torch.randn(2, 37, 64, device="cuda", generator=torch.Generator("cuda").manual_seed(4)).to(dtype)
    m64 = copy.deepcopy(m).double()
    x64, res64 = x.double().requires_grad_(), res.double().requires_grad_()
    want = reference_layer(m64, x64, res64)
    with torch.no_grad():
        assert rel(m(x, residual=res), want) <= tol
        assert rel(m(x), reference_layer(m64, x64)) <= tol
    xs, rs = x.clone().requires_grad_(), res.clone().requires_grad_()
    y = m(xs, residual=rs)
    assert rel(y, want) <= tol
    names, ps = zip(*m.named_parameters())
    got = torch.autograd.grad(y, [xs, rs, *ps], dy)
    ref = torch.autograd.grad(want, [x64, res64, *m64.parameters()], dy.double())
    for n, a, b in zip(("x", "residual", *names), got, ref):
        assert rel(a, b) <= 2 * tol, (n, rel(a, b))


def test_layer_decodes_what_it_prefills():
    m = make(torch.bfloat16).eval()
    x = torch.randn(3, 21, 64, device="cuda", generator=torch.Generator("cuda").manual_seed(5)).bfloat16()
    with torch.no_grad():
        want = m(x)
        cache = GDNCache()
        ys = [m(x[:, :10], cache)]
        ys += [m(x[:, t:t + 1], cache) for t in range(10, 20)]
        ys.append(m(x[:, 20:], cache))
    assert cache.seen == 21 and cache.state.shape == (3, 128, 16)
    assert rel(torch.cat(ys, 1), want) <= 1e-2


def test_fused_mlp():
    for act in ("silu", "gelu"):
        torch.manual_seed(7)
        m = FusedMLP(64, 4.0, act).cuda().bfloat16()
        m64 = copy.deepcopy(m).double()
        x = torch.randn(5, 9, 64, device="cuda").bfloat16().requires_grad_()
        x64 = x.detach().double().requires_grad_()
        f = F.silu if act == "silu" else F.gelu
        want = F.linear(f(F.linear(x64, m64.up.weight, m64.up.bias)), m64.down.weight, m64.down.bias) + x64
        y = m(x, residual=x)
        assert rel(y, want) <= 1e-2
        got = torch.autograd.grad(y.sum(), [x, *m.parameters()])
        ref = torch.autograd.grad(want.sum(), [x64, *m64.parameters()])
        for a, b in zip(got, ref):
            assert rel(a, b) <= 2e-2


def small_lm(**kw):
    torch.manual_seed(11)
    return LM(arch="ssm", d_model=128, n_layer=2, vocab_size=256, mlp_ratio=2.0, mlp="gelu", init_std=0.1, **kw).cuda().bfloat16()


def test_lm_greedy_decoding_and_graph():
    m = small_lm().eval()
    idx = torch.randint(0, 256, (4, 30), device="cuda", generator=torch.Generator("cuda").manual_seed(6))
    ids, got = greedy_decode(m, idx, 8, return_logits=True)
    ids_g, got_g = greedy_decode(m, idx, 8, return_logits=True, graph=True)
    assert torch.equal(ids, ids_g) and torch.equal(got, got_g)  # the same kernels, replayed
    with torch.no_grad():
        full = m(ids[:, :-1])[0][:, 29:]
    assert rel(got, full) <= 2e-2
    with bind_caches(m) as caches:
        assert len(caches) == 2


def test_lm_trains():
    m = small_lm()
    opt = torch.optim.SGD(m.parameters(), lr=0.1)
    idx = torch.randint(0, 256, (8, 65), device="cuda", generator=torch.Generator("cuda").manual_seed(8))
    losses = []
    for _ in range(20):
        opt.zero_grad()
        _, loss = m(idx[:, :-1], idx[:, 1:])
        loss.backward()
        opt.step()
        losses.append(loss.item())
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in m.parameters())
    assert losses[-1] < 0.8 * losses[0], losses


def test_lm_under_compile():
    m = small_lm().eval()
    idx = torch.randint(0, 256, (2, 24), device="cuda", generator=torch.Generator("cuda").manual_seed(9))
    with torch.no_grad():
        want = m(idx)[0]
        got = torch.compile(m, dynamic=False)(idx)[0]
    assert rel(got, want) <= 2e-2
