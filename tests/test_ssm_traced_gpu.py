"""The operators where a call is traced: torch.compile without graph breaks, torch.export and torch.jit.trace give what
the plain calls give (the same kernels, so bitwise where nothing else is between)."""

import copy

import pytest
import torch

from archbench_b200 import ops, traced_ops
from archbench_b200.layers import GDNCache
from archbench_b200.lm import LM
from archbench_b200.ssm_layer import FusedMLP, SelectiveSSM

pytestmark = pytest.mark.gpu


def rnd(seed, *s, dtype=torch.float32):
    return torch.randn(*s, generator=torch.Generator("cuda").manual_seed(seed), device="cuda").to(dtype)


def inputs(dtype, grad=False):
    """Named arguments of each operator, with absent ones, odd views and other types among them."""
    x, z, dt = rnd(1, 2, 9, 48, dtype=dtype)[..., :24], rnd(2, 2, 9, 24, dtype=dtype), rnd(3, 2, 9, 24, dtype=dtype)
    A, D, b = -torch.rand(24, 8, device="cuda") - 0.1, rnd(4, 24), rnd(5, 24)
    Bm, C, h = rnd(6, 2, 9, 8, dtype=dtype), rnd(7, 2, 9, 2, 4 * 2, dtype=dtype)[:, :, :1], rnd(8, 2, 24, 8)
    n = torch.tensor([9, 4], device="cuda")
    conv = [dict(x=x, weight=rnd(9, 24, 1, 4, dtype=dtype), bias=rnd(10, 24), activation="silu", initial_state=rnd(11, 2, 24, 3), output_final_state=True, lengths=n),
            dict(x=x, weight=rnd(9, 24, 3))]
    scan = [dict(x=x, dt=dt, A=A, B=Bm, C=C, D=D, z=z, dt_bias=b, dt_softplus=True, initial_state=h, output_final_state=True, lengths=n),
            dict(x=x, dt=dt, A=A, B=Bm, C=C, dt_softplus=True)]
    xb, w = rnd(12, 3, 5, 40, dtype=torch.bfloat16), rnd(13, 24, 40, dtype=torch.bfloat16)
    lin = [dict(x=xb, weight=w, bias=rnd(14, 24, dtype=torch.bfloat16), activation="gelu", residual=rnd(15, 3, 5, 24, dtype=torch.bfloat16)),
           dict(x=xb, weight=w)]
    return [("causal_conv", a) for a in conv] + [("selective_scan", a) for a in scan] + [("linear", a) for a in lin]


def run(name, fn, kw, grad):
    """Outputs and, with ``grad``, the gradients of every floating input."""
    own = {k: v.detach().clone().requires_grad_(grad) if torch.is_tensor(v) and v.is_floating_point() else v for k, v in kw.items()}
    out = fn(**own)
    out = [t for t in (out if isinstance(out, tuple) else (out,)) if t is not None]
    if not grad:
        return out
    leaves = [v for v in own.values() if torch.is_tensor(v) and v.requires_grad]
    return out + list(torch.autograd.grad(out, leaves, [rnd(20 + i, *t.shape, dtype=t.dtype) for i, t in enumerate(out)]))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("grad", [False, True])
def test_compiled_calls_equal_plain_ones(dtype, grad):
    for name, kw in inputs(dtype):
        fn = getattr(ops, name)
        torch._dynamo.reset()
        want = run(name, fn, kw, grad)
        got = run(name, torch.compile(fn, fullgraph=True, dynamic=False), kw, grad)
        assert len(got) == len(want)
        for i, (a, b) in enumerate(zip(got, want)):
            assert a.dtype == b.dtype and torch.equal(a, b), (name, i)


def test_registrations():
    """Schemas, autograd and fake forms agree with what the operators do."""
    checks = ("test_schema", "test_autograd_registration", "test_faketensor")
    for dtype in (torch.float32, torch.bfloat16):
        for name, kw in inputs(dtype):
            ref = {k: v.detach().clone().requires_grad_() if torch.is_tensor(v) and v.is_floating_point() else v for k, v in kw.items()}
            seen = []
            op = {"causal_conv": "_conv", "selective_scan": "_scan", "linear": "_linear"}[name]
            real = getattr(traced_ops, op)

            class Spy:
                def __call__(self, *a):
                    seen.append(a)
                    return real(*a)

            setattr(traced_ops, op, Spy())
            try:
                getattr(traced_ops, name)(**ref)
            finally:
                setattr(traced_ops, op, real)
            torch.library.opcheck(real, tuple(t.detach().requires_grad_() if torch.is_tensor(t) and t.requires_grad else t for t in seen[0]),
                                  test_utils=checks)


def test_compiled_one_token_forms():
    x, w, A, B = rnd(1, 2, 8), rnd(2, 8, 4), -torch.ones(8, 4, device="cuda"), rnd(3, 2, 4)
    states = [(torch.zeros(2, 8, 3, device="cuda"), torch.zeros(2, 8, 4, device="cuda")) for _ in range(2)]

    def step(x, sc, ss):
        u = ops.causal_conv_step(x, w, sc, activation="silu")
        return ops.selective_scan_step(u, u, A, B, B, ss, dt_softplus=True)

    compiled = torch.compile(step, fullgraph=True, dynamic=False)
    with torch.no_grad():
        for i in range(3):
            assert torch.equal(step(x + i, *states[0]), compiled(x + i, *states[1]))
    for a, b in zip(*states):
        assert torch.equal(a, b) and a.abs().sum() > 0


@pytest.mark.parametrize("train", [False, True])
def test_language_model_compiles_whole(train):
    """Relative error in the 2-norm against the eager model: bf16 elementwise work fused and reordered around the same
    kernels, a few roundings of 2^-9 each per layer: 2e-2, as for the eager model against 64 bits."""
    torch.manual_seed(3)
    m = LM(arch="ssm", d_model=128, n_layer=2, vocab_size=256, mlp_ratio=2.0, mlp="gelu", init_std=0.1).cuda().bfloat16()
    other = copy.deepcopy(m)
    idx = torch.randint(0, 256, (2, 25), device="cuda", generator=torch.Generator("cuda").manual_seed(9))
    torch._dynamo.reset()
    compiled = torch.compile(other, fullgraph=True, dynamic=False)
    rel = lambda a, b: ((a.double() - b.double()).norm() / b.double().norm()).item()
    if not train:
        with torch.no_grad():
            assert rel(compiled(idx)[0], m(idx)[0]) <= 2e-2
        return
    _, want = m(idx[:, :-1], idx[:, 1:])
    _, got = compiled(idx[:, :-1], idx[:, 1:])
    assert rel(got.detach(), want.detach()) <= 2e-2
    want.backward()
    got.backward()
    for (n, a), b in zip(m.named_parameters(), other.parameters()):
        assert rel(b.grad, a.grad) <= 4e-2, (n, rel(b.grad, a.grad))


@pytest.mark.parametrize("make", [lambda: SelectiveSSM(64), lambda: FusedMLP(64, 2.0, "silu")])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_traced_and_exported_layers(make, dtype):
    torch.manual_seed(4)
    m = make().cuda().to(dtype).eval()
    x, other = rnd(1, 2, 11, 64, dtype=dtype), rnd(2, 2, 11, 64, dtype=dtype)
    with torch.no_grad():
        want = [m(x), m(other)]
        traced = torch.jit.trace(m, (x,), check_trace=False)
        for a, b in zip((traced(x), traced(other)), want):
            assert torch.equal(a, b)
        exported = torch.export.export(m, (x,)).module()
        for a, b in zip((exported(x), exported(other)), want):
            assert torch.equal(a, b)


def test_plain_calls_after_tracing_keep_their_parameters():
    """What is derived from a parameter for plain calls follows the parameter, traced calls between or not."""
    torch.manual_seed(5)
    m = SelectiveSSM(64).cuda().eval()
    x = rnd(1, 2, 5, 64)
    with torch.no_grad():
        torch.compile(m, fullgraph=True, dynamic=False)(x)
        before = m(x)
        m.D.add_(1)
        after = m(x)
        cache = GDNCache()
        again = torch.cat([m(x[:, :3], cache), m(x[:, 3:4], cache), m(x[:, 4:], cache)], 1)
    assert not torch.equal(before, after)
    assert ((again - after).norm() <= 1e-5 * after.norm()).item()


def test_traced_calls_refuse_what_plain_ones_refuse():
    """Shapes that the registered forms bring to their own first: a mismatch must not be reshaped away."""
    x, w = rnd(1, 4, 16, dtype=torch.bfloat16), rnd(2, 8, 16, dtype=torch.bfloat16)
    c, k = rnd(3, 2, 5, 8), rnd(4, 8, 2, 4)
    bad = [("linear", (x, w[:, :8])), ("linear", (x, w, None, None, rnd(5, 8, 4, dtype=torch.bfloat16))), ("linear", (x, w[0])),
           ("linear", (x.float(), w.float())), ("linear", (x, w, None, "relu")), ("causal_conv", (c, k)), ("causal_conv", (c, k[:, 0], None, "gelu")),
           ("selective_scan", (c, c[:, :3], -rnd(6, 8, 4).abs(), c[..., :4], c[..., :4]))]
    for name, args in bad:
        for fn in (getattr(ops, name), getattr(traced_ops, name)):
            with pytest.raises(ValueError):
                fn(*args)


@pytest.mark.parametrize("B,T", [(0, 5), (2, 0)])
def test_traced_calls_without_tokens(B, T):
    """No outputs to compute, but gradients that pass through: of the state as its own tensor, zeros for the rest."""
    for m in (ops, traced_ops):
        x, w, s = (torch.zeros(*shape, device="cuda", requires_grad=True) for shape in ((B, T, 8), (8, 4), (B, 8, 3)))
        y, last = m.causal_conv(x, w, None, "silu", s, True)
        d = torch.full_like(last, 2.0)
        gx, gw, gs = torch.autograd.grad([y, last], [x, w, s], [torch.zeros_like(y), d])
        assert gx.shape == x.shape and torch.equal(gw, torch.zeros_like(w)) and torch.equal(gs, d)
        A, h = -torch.ones(8, 4, device="cuda"), torch.zeros(B, 8, 4, device="cuda", requires_grad=True)
        Bm = torch.zeros(B, T, 4, device="cuda")
        y, last = m.selective_scan(x, x, A, Bm, Bm, initial_state=h, output_final_state=True)
        d = torch.full_like(last, 3.0)
        gx, gh = torch.autograd.grad([y, last], [x, h], [torch.zeros_like(y), d])
        assert gx.shape == x.shape and torch.equal(gh, d)
        v, wl = torch.zeros(B * T, 16, device="cuda", dtype=torch.bfloat16, requires_grad=True), torch.ones(8, 16, device="cuda", dtype=torch.bfloat16, requires_grad=True)
        gv, gw = torch.autograd.grad(m.linear(v, wl, None, "gelu").sum(), [v, wl])
        assert gv.shape == v.shape and torch.equal(gw, torch.zeros_like(wl))
