"""The selective-state-space operators on the GPU against plain 64-bit forms: outputs, final states and gradients, at the
sizes, strides and row lengths where the kernels change path."""

import pytest
import torch

from archbench_b200 import ops
import ssm_reference as R

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def rnd(g, *s):
    return torch.randn(*s, generator=g, device="cuda")


def wide(t, pad):
    """The same values as a view with odd row strides and a start that no vector load can take (pad > 0)."""
    if not pad:
        return t
    big = torch.full((*t.shape[:-1], t.shape[-1] + 2 * pad + 1), float("nan"), device=t.device, dtype=t.dtype)
    big[..., pad:pad + t.shape[-1]] = t
    return big[..., pad:pad + t.shape[-1]]


def lens(B, T, g):
    n = torch.randint(0, T + 1, (B,), generator=g, device="cuda")
    n[0] = T
    if B > 1:
        n[1] = 0
    return n


# ---- convolution ------------------------------------------------------------------------------

CONV = [  # B, T, C, W, dtype, silu, bias, state, lengths, pad
    (1, 1, 1, 2, "f32", True, True, True, False, 0),
    (2, 3, 8, 4, "bf16", True, True, True, True, 0),
    (2, 16, 64, 4, "bf16", True, True, False, False, 0),
    (3, 17, 24, 3, "f32", False, False, True, True, 0),
    (2, 50, 40, 4, "bf16", True, True, True, True, 3),
    (2, 49, 37, 4, "f32", True, False, True, True, 1),
    (4, 33, 128, 2, "bf16", False, True, False, True, 0),
    (3, 131, 256, 4, "bf16", True, True, True, True, 0),
]


def conv_case(B, T, C, W, dtype, silu, bias, state, lengths, pad):
    g = torch.Generator("cuda").manual_seed(B * 1000 + T * 10 + C)
    dt = DT[dtype]
    v = dict(x=rnd(g, B, T, C).to(dt), weight=rnd(g, C, W).to(dt), bias=rnd(g, C).to(dt) if bias else None,
             state=rnd(g, B, C, W - 1).to(dt) if state else None)
    return v, lens(B, T, g) if lengths else None, rnd(g, B, T, C).to(dt), rnd(g, B, C, W - 1).to(dt)


@pytest.mark.parametrize("case", CONV)
def test_conv_forward_and_backward(case):
    B, T, C, W, dtype, silu, bias, state, lengths, pad = case
    v, n, dy, dlast = conv_case(*case)
    ref = {k: None if t is None else t.double().cpu().requires_grad_() for k, t in v.items()}
    y0, last0 = R.conv(ref["x"], ref["weight"], ref["bias"], silu, ref["state"], n)
    own = {k: None if t is None else t.clone().requires_grad_() for k, t in v.items()}
    act = "silu" if silu else None
    with torch.no_grad():
        y, last = ops.causal_conv(wide(v["x"], pad), v["weight"], v["bias"], act, v["state"], True, n)
    R.close(y, y0, "y")
    assert torch.equal(last.double().cpu(), last0.detach())
    y, last = ops.causal_conv(wide(own["x"], pad), own["weight"][:, None], own["bias"], act, own["state"], True, n)
    names = [k for k in own if own[k] is not None]
    got = torch.autograd.grad([y, last], [own[k] for k in names], [wide(dy, pad), dlast])
    want = torch.autograd.grad([y0, last0], [ref[k] for k in names], [dy.double().cpu(), dlast.double().cpu()])
    for k, a, b in zip(names, got, want):
        R.close(a, b, "d" + k, accumulated=64 + B * T)


def test_conv_step_continues_the_prompt():
    for dtype, C, W in (("bf16", 64, 4), ("f32", 37, 3), ("bf16", 19, 2)):
        v, _, _, _ = conv_case(3, 12, C, W, dtype, True, True, True, False, 0)
        want, wlast = ops.causal_conv(v["x"], v["weight"], v["bias"], "silu", v["state"], True)
        state = v["state"].clone()
        ys = [ops.causal_conv_step(v["x"][:, t], v["weight"], state, v["bias"], "silu") for t in range(12)]
        assert torch.equal(torch.stack(ys, 1), want) and torch.equal(state, wlast)


def test_conv_pieces_equal_the_whole():
    v, _, _, _ = conv_case(2, 64, 64, 4, "bf16", True, True, True, False, 0)
    want, wlast = ops.causal_conv(v["x"], v["weight"], v["bias"], "silu", v["state"], True)
    st, ys = v["state"], []
    for a, b in ((0, 0), (0, 1), (1, 3), (3, 40), (40, 64)):
        y, st = ops.causal_conv(v["x"][:, a:b], v["weight"], v["bias"], "silu", st, True)
        ys.append(y)
    assert torch.equal(torch.cat(ys, 1), want) and torch.equal(st, wlast)


# ---- scan -------------------------------------------------------------------------------------

SCAN = [  # B, T, D, N, G, dtype, gate, skip, bias, softplus, state, lengths, pad
    (1, 1, 1, 1, 1, "f32", True, True, True, True, True, False, 0),
    (2, 1, 40, 16, 1, "bf16", True, True, True, True, True, True, 0),
    (2, 31, 64, 16, 2, "bf16", True, True, True, True, True, True, 0),
    (1, 32, 33, 4, 1, "f32", False, False, False, False, False, False, 0),
    (3, 45, 48, 5, 3, "f32", True, True, True, True, True, True, 2),
    (2, 70, 30, 24, 2, "f32", False, True, True, True, True, True, 1),
    (2, 65, 20, 64, 1, "bf16", True, True, True, True, False, True, 0),
    (2, 48, 130, 8, 1, "bf16", False, True, False, True, True, False, 3),
    (1, 300, 40, 16, 1, "f32", True, True, True, True, True, False, 0),   # split over time
    (2, 530, 24, 16, 2, "f32", True, True, True, True, True, True, 0),    # split, ragged
    (1, 1100, 16, 33, 1, "bf16", True, True, True, True, False, False, 0),
    # rows that 16-byte copies take, each layout of lanes, tiles cut by lengths, ends and channel blocks
    (3, 37, 144, 8, 1, "bf16", True, True, True, True, True, True, 0),
    (2, 50, 260, 4, 1, "f32", True, True, True, True, True, True, 0),
    (3, 41, 72, 16, 3, "bf16", False, False, True, True, True, True, 0),
    (2, 33, 80, 16, 2, "f32", True, True, True, True, True, False, 0),
    (2, 40, 48, 16, 1, "f32", True, True, False, False, True, True, 0),
    (2, 57, 48, 24, 1, "bf16", True, True, True, True, True, True, 0),
    (2, 35, 40, 32, 1, "f32", True, True, False, True, True, True, 0),
    (2, 43, 24, 64, 1, "bf16", True, True, True, True, True, True, 0),
    (2, 29, 28, 48, 1, "f32", False, True, True, True, True, True, 0),
    (1, 700, 32, 16, 1, "bf16", True, True, True, True, True, True, 0),
    # odd widths and rows off their boundaries: laid out again first
    (2, 45, 57, 16, 3, "bf16", True, True, True, True, True, True, 0),
    (2, 300, 21, 4, 1, "bf16", True, True, True, True, True, True, 3),
    (1, 200, 35, 24, 5, "f32", True, True, True, True, True, False, 1),
    (2, 50, 67, 64, 1, "f32", False, True, True, True, True, True, 0),
    (2, 40, 31, 8, 1, "f32", True, False, True, True, False, True, 2),
]


def scan_case(B, T, D, N, G, dtype, gate, skip, bias, softplus, state, lengths, pad):
    g = torch.Generator("cuda").manual_seed(B * 1000 + T * 10 + D + N)
    dt = DT[dtype]
    step = rnd(g, B, T, D)
    v = dict(x=rnd(g, B, T, D).to(dt), dt=(step if softplus else 0.2 * step.abs()).to(dt),
             A=-torch.rand(D, N, generator=g, device="cuda") * 4 - 0.01, B=rnd(g, B, T, G, N).to(dt), C=rnd(g, B, T, G, N).to(dt),
             D=rnd(g, D) if skip else None, z=rnd(g, B, T, D).to(dt) if gate else None, dt_bias=rnd(g, D) - 2 if bias else None,
             state=rnd(g, B, D, N) if state else None)
    return v, lens(B, T, g) if lengths else None, rnd(g, B, T, D).to(dt), rnd(g, B, D, N)


def run_own(v, softplus, n, pad=0):
    w = lambda k: None if v[k] is None else wide(v[k], pad)
    return ops.selective_scan(w("x"), w("dt"), v["A"], w("B"), w("C"), D=v["D"], z=w("z"), dt_bias=v["dt_bias"],
                              dt_softplus=softplus, initial_state=v["state"], output_final_state=True, lengths=n)


def run_ref(v, softplus, n):
    return R.scan(v["x"], v["dt"], v["A"], v["B"], v["C"], v["D"], v["z"], v["dt_bias"], softplus, v["state"], n)


@pytest.mark.parametrize("case", SCAN)
def test_scan_forward_and_backward(case):
    B, T, D, N, G, dtype, gate, skip, bias, softplus, state, lengths, pad = case
    v, n, dy, dlast = scan_case(*case)
    ref = {k: None if t is None else t.double().cpu().requires_grad_() for k, t in v.items()}
    y0, last0 = run_ref(ref, softplus, n)
    with torch.no_grad():
        y, last = run_own(v, softplus, n, pad)
    # a value passes through at most T decays, each with a few roundings, of which the far ones are damped
    R.close(y, y0, "y", accumulated=128 + N)
    R.close(last, last0, "state", accumulated=128)
    own = {k: None if t is None else t.clone().requires_grad_() for k, t in v.items()}
    y, last = run_own(own, softplus, n, pad)
    names = [k for k in own if own[k] is not None]
    got = torch.autograd.grad([y, last], [own[k] for k in names], [wide(dy, pad), dlast])
    want = torch.autograd.grad([y0, last0], [ref[k] for k in names], [dy.double().cpu(), dlast.double().cpu()])
    for k, a, b in zip(names, got, want):
        R.close(a, b, "d" + k, accumulated=256 + (B * T if k in ("A", "D", "dt_bias") else D // G if k in "BC" else 0))


def test_scan_gradient_against_differences():
    """The kernel's own outputs, moved along a random direction of every input."""
    case = (2, 40, 24, 16, 2, "f32", True, True, True, True, True, True, 0)
    v, n, dy, dlast = scan_case(*case)
    own = {k: t.clone().requires_grad_() for k, t in v.items()}
    y, last = run_own(own, True, n)
    grads = torch.autograd.grad([y, last], list(own.values()), [dy, dlast])
    g = torch.Generator("cuda").manual_seed(5)
    eps = 2.0 ** -9
    for (k, t), gr in zip(v.items(), grads):
        d = rnd(g, *t.shape)
        def loss(sign):
            with torch.no_grad():
                a, b = run_own({**v, k: t + sign * eps * d}, True, n)
            return (a.double() * dy.double()).sum() + (b.double() * dlast.double()).sum()
        diff = ((loss(1) - loss(-1)) / (2 * eps)).item()
        dot = (gr.double() * d.double()).sum().item()
        # third derivatives times eps^2, and the outputs' fp32 roundings over eps: a few parts in a thousand of the
        # gradient's size along a direction
        scale = (gr.double().norm()).item()
        assert abs(diff - dot) <= 5e-3 * scale + 1e-3, (k, diff, dot, scale)


def test_scan_step_continues_the_prompt():
    for case in ((3, 9, 40, 16, 2, "bf16", True, True, True, True, True, False, 0), (2, 9, 21, 5, 1, "f32", False, True, False, True, True, False, 0),
                 (1, 9, 6, 64, 3, "f32", True, False, True, True, True, False, 0)):
        v, _, _, _ = scan_case(*case)
        want, last0 = run_ref({k: None if t is None else t.double().cpu() for k, t in v.items()}, True, None)
        state = v["state"].clone()
        for t in range(9):
            at = lambda k: None if v[k] is None else v[k][:, t]
            y = ops.selective_scan_step(at("x"), at("dt"), v["A"], at("B"), at("C"), state, D=v["D"], z=at("z"), dt_bias=v["dt_bias"], dt_softplus=True)
            R.close(y, want[:, t], f"y{t}", accumulated=128)
        R.close(state, last0, "state", accumulated=128)


def test_scan_pieces_equal_the_whole():
    case = (2, 96, 40, 16, 1, "f32", True, True, True, True, True, False, 0)
    v, _, _, _ = scan_case(*case)
    want, wlast = run_own(v, True, None)
    st, ys = v["state"], []
    for a, b in ((0, 0), (0, 1), (1, 33), (33, 96)):
        cut = {k: t[:, a:b] if k in ("x", "dt", "B", "C", "z") else t for k, t in v.items()}
        y, st = run_own({**cut, "state": st}, True, None)
        ys.append(y)
    assert torch.equal(torch.cat(ys, 1), want) and torch.equal(st, wlast)


def test_scan_masked_places_are_not_read():
    """Whatever stands past a row's length -- NaN and infinities too -- reaches no output and no gradient."""
    case = (3, 80, 40, 16, 1, "f32", True, True, True, True, True, True, 0)
    v, n, dy, dlast = scan_case(*case)
    bad = {k: t.clone() for k, t in v.items()}
    dyb = dy.clone()
    for b in range(3):
        for k, w in (("x", float("nan")), ("dt", float("inf")), ("B", float("nan")), ("C", float("-inf")), ("z", float("nan"))):
            bad[k][b, int(n[b]):] = w
        dyb[b, int(n[b]):] = float("nan")
    outs = []
    for vals, d in ((v, dy), (bad, dyb)):
        own = {k: t.clone().requires_grad_() for k, t in vals.items()}
        y, last = run_own(own, True, n)
        outs.append([y, last, *torch.autograd.grad([y, last], list(own.values()), [d, dlast])])
    for a, b in zip(*outs):
        assert torch.equal(a, b) and torch.isfinite(a).all()


def test_scan_large_steps_and_saturated_inputs():
    """Step sizes past softplus's linear knee forget the state at once; tiny ones keep it; no overflow either way."""
    g = torch.Generator("cuda").manual_seed(1)
    x, B, C = rnd(g, 1, 40, 8), rnd(g, 1, 40, 1, 16), rnd(g, 1, 40, 1, 16)
    A = -torch.rand(8, 16, generator=g, device="cuda") * 16 - 1
    for raw in (90.0, -90.0, 0.0):
        dt = torch.full((1, 40, 8), raw, device="cuda")
        h0 = rnd(g, 1, 8, 16)
        y, last = ops.selective_scan(x, dt, A, B, C, dt_softplus=True, initial_state=h0, output_final_state=True)
        c = lambda t: t.double().cpu()
        y0, l0 = R.scan(c(x), c(dt), c(A), c(B), c(C), softplus=True, state=c(h0))
        R.close(y, y0, f"y at {raw}", accumulated=128)
        R.close(last, l0, f"state at {raw}", accumulated=128)


def test_scan_is_deterministic_and_on_any_stream():
    case = (2, 530, 24, 16, 2, "bf16", True, True, True, True, True, True, 0)
    v, n, dy, dlast = scan_case(*case)
    runs = []
    for s in (torch.cuda.current_stream(), torch.cuda.Stream()):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            own = {k: t.clone().requires_grad_() for k, t in v.items()}
            y, last = run_own(own, True, n)
            grads = torch.autograd.grad([y, last], list(own.values()), [dy, dlast])
        torch.cuda.current_stream().wait_stream(s)
        torch.cuda.synchronize()
        runs.append([y, last, *grads])
    for a, b in zip(*runs):
        assert torch.equal(a, b)


def test_empty_batches_and_sequences():
    for B, T in ((0, 5), (2, 0)):
        x = torch.zeros(B, T, 8, device="cuda", requires_grad=True)
        Bm = torch.zeros(B, T, 4, device="cuda")
        A = -torch.ones(8, 4, device="cuda")
        h0 = torch.ones(B, 8, 4, device="cuda", requires_grad=True)
        y, last = ops.selective_scan(x, x, A, Bm, Bm, initial_state=h0, output_final_state=True)
        assert y.shape == x.shape and torch.equal(last, h0)
        gx, gh = torch.autograd.grad([y, last], [x, h0], [y, torch.full_like(last, 2.0)])
        assert gx.shape == x.shape and torch.equal(gh, torch.full_like(h0, 2.0))
        st = torch.ones(B, 8, 3, device="cuda")
        y, last = ops.causal_conv(x.detach(), torch.ones(8, 4, device="cuda"), initial_state=st, output_final_state=True)
        assert y.shape == x.shape and torch.equal(last, st)


def test_refusals():
    x = torch.zeros(2, 4, 8, device="cuda")
    A, Bm, w = -torch.ones(8, 4, device="cuda"), torch.zeros(2, 4, 4, device="cuda"), torch.zeros(8, 4, device="cuda")
    bad = [
        lambda: ops.selective_scan(x.cpu(), x, A, Bm, Bm),
        lambda: ops.selective_scan(x.half(), x, A, Bm, Bm),
        lambda: ops.selective_scan(x[0], x, A, Bm, Bm),
        lambda: ops.selective_scan(x, x[:, :3], A, Bm, Bm),
        lambda: ops.selective_scan(x, x, A[:4], Bm, Bm),
        lambda: ops.selective_scan(x, x, -torch.ones(8, 65, device="cuda"), Bm, Bm),
        lambda: ops.selective_scan(x, x, A, Bm[:, :, None].expand(2, 4, 3, 4), Bm[:, :, None].expand(2, 4, 3, 4)),
        lambda: ops.selective_scan(x, x, A, Bm, Bm[..., :3]),
        lambda: ops.selective_scan(x, x, A, Bm, Bm, initial_state=torch.zeros(2, 4, 8, device="cuda")),
        lambda: ops.selective_scan(x, x, A, Bm, Bm, lengths=torch.zeros(3, device="cuda", dtype=torch.int32)),
        lambda: ops.selective_scan(x, x, A, Bm, Bm, lengths=torch.zeros(2, device="cuda")),
        lambda: ops.selective_scan_step(x[:, 0], x[:, 0], A, Bm[:, 0], Bm[:, 0], torch.zeros(2, 8, 4, device="cuda", dtype=torch.bfloat16)),
        lambda: ops.selective_scan_step(x, x, A, Bm, Bm, torch.zeros(2, 8, 4, device="cuda")),
        lambda: ops.causal_conv(x, torch.zeros(8, 5, device="cuda")),
        lambda: ops.causal_conv(x, torch.zeros(7, 4, device="cuda")),
        lambda: ops.causal_conv(x, w, activation="gelu"),
        lambda: ops.causal_conv(x, w, initial_state=torch.zeros(2, 8, 4, device="cuda")),
        lambda: ops.causal_conv_step(x[:, 0], w, torch.zeros(2, 3, 8, device="cuda").transpose(1, 2)),
        lambda: ops.causal_conv_step(x[:, 0].double(), w, torch.zeros(2, 8, 3, device="cuda")),
    ]
    for f in bad:
        with pytest.raises(ValueError):
            f()
