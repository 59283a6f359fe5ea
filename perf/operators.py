"""The workloads by which the selective-state-space mixer's operators and the fused linear layer are timed.

Four operators, as a mixer layer runs them one after the other:

  causal_conv     y_t = act(bias + sum_w weight[:, w] x_{t-W+1+w}), depthwise, channels last
  selective_scan  h_t = exp(s_t A) h_{t-1} + s_t B_t x_t;  y_t = (C_t . h_t + D x_t) silu(z_t)
  *_step          one token of either, the state updated in place
  linear          y = act(x weight^T + bias) + residual

Sizes are those of the package's own configurations (batch 8 x 4096 tokens, 65536 tokens in one sequence,
256 decode streams, model width 1024, SwiGLU hidden 2816) with the mixer at twice the model width, and
generic odd ones.  ``run`` has each operator in plain form (32-bit elementary torch operations, rounded once
at the end) and as a call of the package's operator; ``exact`` restates the definitions in 64 bits, token by
token.
"""

from __future__ import annotations

import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp32": torch.float32}
_DEV = "cuda"


def listed():
    return [
        # A prompt batch through the mixer's short convolution: the first half of the input projection, as a view.
        dict(name="conv prompt 8x4096x2048", op="conv", B=8, T=4096, C=2048, W=4, dtype="bf16", act=True, bias=True, state=True, train=False, ragged=False),
        # A training step of the convolution, forward and backward.
        dict(name="conv train 8x2048x2048", op="conv", B=8, T=2048, C=2048, W=4, dtype="bf16", act=True, bias=True, state=False, train=True, ragged=False),
        # The convolution of one decode step for 256 streams.
        dict(name="conv step 256x2048", op="conv_step", B=256, C=2048, W=4, dtype="bf16", act=True, bias=True),
        # A prompt batch through the scan, gated, final state kept for decoding.
        dict(name="scan prompt 8x4096x2048", op="scan", B=8, T=4096, D=2048, N=16, G=1, dtype="bf16", gate=True, state=False, train=False, ragged=False),
        # One long document: few rows, split over time; continues an earlier state.
        dict(name="scan long 1x65536x2048", op="scan", B=1, T=65536, D=2048, N=16, G=1, dtype="bf16", gate=True, state=True, train=False, ragged=False),
        # A right-padded batch of short prompts in fp32 with two groups and an odd width.
        dict(name="scan ragged 3x777x1002", op="scan", B=3, T=777, D=1002, N=24, G=2, dtype="fp32", gate=False, state=True, train=False, ragged=True),
        # A training step of the scan, forward and backward.
        dict(name="scan train 8x2048x2048", op="scan", B=8, T=2048, D=2048, N=16, G=1, dtype="bf16", gate=True, state=False, train=True, ragged=False),
        # The scan of one decode step for 256 streams: the state is read and written once.
        dict(name="scan step 256x2048", op="scan_step", B=256, D=2048, N=16, G=1, dtype="bf16", gate=True),
        # The mixer's output projection with the block's residual, one decode step of 16 streams.
        dict(name="linear step 16x1024x2048", op="linear", M=16, N=1024, K=2048, bias=False, act="none", residual=True, train=False),
        # An MLP's expanding projection over a prompt batch.
        dict(name="linear prompt 32768x2816x1024", op="linear", M=32768, N=2816, K=1024, bias=True, act="silu", residual=False, train=False),
        # A training step of a biased, activated projection with the residual, forward and backward.
        dict(name="linear train 16384x1024x2816", op="linear", M=16384, N=1024, K=2816, bias=True, act="gelu", residual=True, train=True),
        # A ragged token count and odd widths: rows that no wide load can take.
        dict(name="linear odd 1001x501x999", op="linear", M=1001, N=501, K=999, bias=True, act="gelu", residual=True, train=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["conv", "conv", "conv_step", "scan", "scan", "scan", "scan_step", "linear", "linear", "linear"])
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    if op == "conv":
        C, W = _log(rng, 64, 4096), rng.choice([2, 3, 4])
        B = _log(rng, 1, 16)
        T = _log(rng, 1, max(1, min(16384, 2**25 // (B * C))))
        return dict(op=op, B=B, T=T, C=C, W=W, dtype=dtype, act=rng.random() < 0.8, bias=rng.random() < 0.7,
                    state=rng.random() < 0.5, train=rng.random() < 0.4, ragged=rng.random() < 0.3)
    if op == "conv_step":
        return dict(op=op, B=_log(rng, 1, 512), C=_log(rng, 64, 4096), W=rng.choice([2, 3, 4]), dtype=dtype, act=True,
                    bias=rng.random() < 0.7)
    if op == "scan":
        G = rng.choice([1, 1, 2, 4])
        D = G * _log(rng, 32, 3000 // G)
        N = rng.choice([4, 8, 16, 16, 16, 24, 32, 64])
        B, train = _log(rng, 1, 16), rng.random() < 0.4
        T = _log(rng, 1, max(1, min(16384 if train else 32768, 2 ** (28 if train else 29) // (B * D * N))))
        return dict(op=op, B=B, T=T, D=D, N=N, G=G, dtype=dtype, gate=rng.random() < 0.7, state=rng.random() < 0.5,
                    train=train, ragged=rng.random() < 0.3)
    if op == "scan_step":
        G = rng.choice([1, 1, 2, 4])
        return dict(op=op, B=_log(rng, 1, 512), D=G * _log(rng, 32, 3000 // G), N=rng.choice([4, 8, 16, 16, 24, 32, 64]), G=G,
                    dtype=dtype, gate=rng.random() < 0.7)
    N, K = _log(rng, 48, 4096), _log(rng, 48, 4096)
    if rng.random() < 0.7:  # most projections have widths of whole vectors
        N, K = max(8, N // 8 * 8), max(8, K // 8 * 8)
    train = rng.random() < 0.3
    M = _log(rng, 1, max(1, min(32768, 2 ** (35 if train else 36) // (N * K))))
    return dict(op="linear", M=M, N=N, K=K, bias=rng.random() < 0.6, act=rng.choice(["none", "silu", "gelu"]),
                residual=rng.random() < 0.5, train=train)


# ---- inputs -----------------------------------------------------------------------------------


def _lengths(case, gen):
    """Token counts of a right-padded batch: one full row, the others anything down to an empty one."""
    n = torch.randint(0, case["T"] + 1, (case["B"],), generator=gen, device=_DEV, dtype=torch.int32)
    n[0] = case["T"]
    return n


def prepare(case, seed):
    gen = torch.Generator(_DEV).manual_seed(int(seed))
    rnd = lambda *s: torch.randn(*s, generator=gen, device=_DEV)  # noqa: E731
    uni = lambda *s: torch.rand(*s, generator=gen, device=_DEV)  # noqa: E731
    s, op = {"case": dict(case)}, case["op"]
    if op == "linear":
        M, N, K, dt = case["M"], case["N"], case["K"], torch.bfloat16
        s["x"] = rnd(M, K).to(dt)
        s["weight"] = (rnd(N, K) / math.sqrt(K)).to(dt)
        s["bias"] = (0.5 * rnd(N)).to(dt) if case["bias"] else None
        s["residual"] = rnd(M, N).to(dt) if case["residual"] else None
        s["dy"] = rnd(M, N).to(dt) if case["train"] else None
        return s
    dt = _DT[case["dtype"]]
    if op in ("conv", "conv_step"):
        B, C, W = case["B"], case["C"], case["W"]
        tok = (B, case["T"]) if op == "conv" else (B,)
        s["x"] = rnd(*tok, 2 * C).to(dt)[..., :C]  # the first half of an input projection
        s["weight"] = ((2 * uni(C, W) - 1) / math.sqrt(W)).to(dt)
        s["bias"] = (0.2 * rnd(C)).to(dt) if case["bias"] else None
        s["activation"] = "silu" if case["act"] else None
        if op == "conv_step":
            s["state"] = rnd(B, C, W - 1).to(dt)
            return s
        s["state"] = rnd(B, C, W - 1).to(dt) if case["state"] else None
        s["lengths"] = _lengths(case, gen) if case["ragged"] else None
        s["dy"] = rnd(*tok, C).to(dt) if case["train"] else None
        return s
    B, D, N, G = case["B"], case["D"], case["N"], case["G"]
    tok = (B, case["T"]) if op == "scan" else (B,)
    s["x"] = torch.nn.functional.silu(rnd(*tok, D)).to(dt)
    s["dt"] = (0.5 * rnd(*tok, D)).to(dt)
    R = (D + 15) // 16 * 8
    bc = rnd(*tok, R + 2 * G * N).to(dt)  # the low-rank step sizes, B and C: one projection's output
    s["B"] = bc[..., R:R + G * N].unflatten(-1, (G, N))
    s["C"] = bc[..., R + G * N:].unflatten(-1, (G, N))
    s["z"] = rnd(*tok, 2 * D).to(dt)[..., D:] if case["gate"] else None  # the second half of the input projection
    s["A"] = -torch.arange(1, N + 1, device=_DEV, dtype=torch.float32).expand(D, N) * (0.8 + 0.4 * uni(D, N))
    s["D"] = 1 + 0.1 * rnd(D)
    step = torch.exp(math.log(1e-3) + (math.log(1e-1) - math.log(1e-3)) * uni(D))
    s["dt_bias"] = step + torch.log(-torch.expm1(-step))  # softplus(dt_bias) = step
    if op == "scan_step":
        s["state"] = 0.5 * rnd(B, D, N)
        return s
    s["state"] = 0.5 * rnd(B, D, N) if case["state"] else None
    s["lengths"] = _lengths(case, gen) if case["ragged"] else None
    s["dy"] = rnd(*tok, D).to(dt) if case["train"] else None
    s["dstate"] = rnd(B, D, N) if case["train"] else None
    return s


# ---- one pass ---------------------------------------------------------------------------------


def run(state):
    op = state["case"]["op"]
    return (_OWN if own else _PLAIN)[op](state)


def _named(**kw):
    return {k: v for k, v in kw.items() if v is not None}


def _own_conv(s):
    from archbench_b200 import ops

    c = s["case"]
    if not c["train"]:
        y, last = ops.causal_conv(s["x"], s["weight"], s["bias"], activation=s["activation"], initial_state=s["state"],
                                  output_final_state=True, lengths=s["lengths"])
        return dict(y=y, state=last)
    leaf = {k: s[k].detach().requires_grad_() for k in ("x", "weight", "bias", "state") if s[k] is not None}
    y, _ = ops.causal_conv(leaf["x"], leaf["weight"], leaf.get("bias"), activation=s["activation"], initial_state=leaf.get("state"),
                           lengths=s["lengths"])
    grads = torch.autograd.grad(y, list(leaf.values()), s["dy"])
    return dict(y=y.detach(), **{"d" + k: g for k, g in zip(leaf, grads)})


def _own_conv_step(s):
    from archbench_b200 import ops

    y = ops.causal_conv_step(s["x"], s["weight"], s["state"], s["bias"], activation=s["activation"])
    return dict(y=y, state=s["state"])


def _own_scan(s):
    from archbench_b200 import ops

    if not s["case"]["train"]:
        y, last = ops.selective_scan(s["x"], s["dt"], s["A"], s["B"], s["C"], D=s["D"], z=s["z"], dt_bias=s["dt_bias"],
                                     dt_softplus=True, initial_state=s["state"], output_final_state=True, lengths=s["lengths"])
        return dict(y=y, state=last)
    leaf = {k: s[k].detach().requires_grad_() for k in ("x", "dt", "A", "B", "C", "D", "z", "dt_bias", "state") if s[k] is not None}
    y, last = ops.selective_scan(leaf["x"], leaf["dt"], leaf["A"], leaf["B"], leaf["C"], D=leaf["D"], z=leaf.get("z"),
                                 dt_bias=leaf["dt_bias"], dt_softplus=True, initial_state=leaf.get("state"),
                                 output_final_state=True, lengths=s["lengths"])
    grads = torch.autograd.grad([y, last], list(leaf.values()), [s["dy"], s["dstate"]])
    return dict(y=y.detach(), state=last.detach(), **{"d" + k: g for k, g in zip(leaf, grads)})


def _own_scan_step(s):
    from archbench_b200 import ops

    y = ops.selective_scan_step(s["x"], s["dt"], s["A"], s["B"], s["C"], s["state"], D=s["D"], z=s["z"], dt_bias=s["dt_bias"],
                                dt_softplus=True)
    return dict(y=y, state=s["state"])


def _own_linear(s):
    from archbench_b200 import ops

    act = None if s["case"]["act"] == "none" else s["case"]["act"]
    if not s["case"]["train"]:
        return dict(y=ops.linear(s["x"], s["weight"], s["bias"], activation=act, residual=s["residual"]))
    leaf = {k: s[k].detach().requires_grad_() for k in ("x", "weight", "bias", "residual") if s[k] is not None}
    y = ops.linear(leaf["x"], leaf["weight"], leaf.get("bias"), activation=act, residual=leaf.get("residual"))
    grads = torch.autograd.grad(y, list(leaf.values()), s["dy"])
    return dict(y=y.detach(), **{"d" + k: g for k, g in zip(leaf, grads)})


_OWN = dict(conv=_own_conv, conv_step=_own_conv_step, scan=_own_scan, scan_step=_own_scan_step, linear=_own_linear)


# ---- plain forms: 32-bit elementary operations ------------------------------------------------


def _f(t):
    return None if t is None else t.float()


def _silu(x):
    return x * torch.sigmoid(x)


def _dsilu(x):
    g = torch.sigmoid(x)
    return g * (1 + x * (1 - g))


def _softplus(x):
    return torch.clamp(x, min=0) + torch.log1p(torch.exp(-torch.abs(x)))


def _valid(s, x):
    """(B, T, 1): whether a token belongs to its row."""
    return None if s.get("lengths") is None else torch.arange(x.shape[1], device=x.device)[None, :, None] < s["lengths"][:, None, None]


def _windows(s, x, w):
    """(B, C, W, T) views of the padded input, and the padded input (B, C, T + W - 1)."""
    B, T, C = x.shape
    W = w.shape[1]
    past = x.new_zeros(B, C, W - 1) if s["state"] is None else _f(s["state"])
    xp = torch.cat([past, x.transpose(1, 2)], 2)
    return xp.unfold(2, T, 1), xp


def _plain_conv(s):
    x, w, dt = _f(s["x"]), _f(s["weight"]), s["x"].dtype
    B, T, C = x.shape
    W = w.shape[1]
    win, xp = _windows(s, x, w)
    pre = (win * w[None, :, :, None]).sum(2).transpose(1, 2)
    if s["bias"] is not None:
        pre = pre + _f(s["bias"])
    y = _silu(pre) if s["activation"] else pre
    ok = _valid(s, x)
    if ok is not None:
        y = torch.where(ok, y, torch.zeros_like(y))
    if not s["case"]["train"]:
        end = torch.full((B,), T, device=x.device) if s["lengths"] is None else s["lengths"].long()
        at = end[:, None, None] + torch.arange(W - 1, device=x.device)
        return dict(y=y.to(dt), state=torch.gather(xp, 2, at.expand(B, C, W - 1)).to(dt))
    dpre = _f(s["dy"]) * (_dsilu(pre) if s["activation"] else 1.0)
    if ok is not None:
        dpre = torch.where(ok, dpre, torch.zeros_like(dpre))
    dp = dpre.transpose(1, 2)
    dw = (win * dp[:, :, None]).sum((0, 3))
    padded = torch.nn.functional.pad(dp, (W - 1, W - 1))
    dxp = (padded.unfold(2, T + W - 1, 1) * w.flip(1)[None, :, :, None]).sum(2)
    return dict(y=y.to(dt), dx=dxp[:, :, W - 1:].transpose(1, 2).to(dt), dweight=dw.to(dt), **_named(
        dbias=None if s["bias"] is None else dpre.sum((0, 1)).to(dt),
        dstate=None if s["state"] is None else dxp[:, :, :W - 1].to(dt)))


def _plain_conv_step(s):
    x, w, st = _f(s["x"]), _f(s["weight"]), s["state"]
    full = torch.cat([_f(st), x[:, :, None]], 2)
    pre = (full * w).sum(2)
    if s["bias"] is not None:
        pre = pre + _f(s["bias"])
    st.copy_(full[:, :, 1:])
    return dict(y=(_silu(pre) if s["activation"] else pre).to(s["x"].dtype), state=st)


def _prefix(a, b):
    """h_t = a_t h_{t-1} + b_t over dimension 1 from zero, in place in b, by doubling the span that each entry covers."""
    span = 1
    while span < a.shape[1]:
        b[:, span:] = b[:, span:] + a[:, span:] * b[:, :-span]
        a[:, span:] = a[:, span:] * a[:, :-span]
        span *= 2
    return b


def _groups(t, D):
    """(..., G, N) -> (..., D, N): each group's row for its channels."""
    return t.repeat_interleave(D // t.shape[-2], dim=-2)


def _plain_scan(s):
    x, raw, A = _f(s["x"]), _f(s["dt"]) + s["dt_bias"], s["A"]
    D, dt = x.shape[-1], s["x"].dtype
    Bm, Cm, z = _groups(_f(s["B"]), D), _groups(_f(s["C"]), D), _f(s["z"])
    ok = _valid(s, x)
    st = _softplus(raw)
    if ok is not None:
        st = torch.where(ok, st, torch.zeros_like(st))
    a = torch.exp(st[..., None] * A)
    u = (st * x)[..., None] * Bm
    if s["state"] is not None:
        u[:, 0] += a[:, 0] * s["state"]
    h = _prefix(a.clone() if s["case"]["train"] else a, u)
    core = (h * Cm).sum(-1) + s["D"] * x
    y = core if z is None else core * _silu(z)
    if ok is not None:
        y = torch.where(ok, y, torch.zeros_like(y))
    last = h[:, -1].clone()
    if not s["case"]["train"]:
        return dict(y=y.to(dt), state=last)
    dy = _f(s["dy"])
    if ok is not None:
        dy = torch.where(ok, dy, torch.zeros_like(dy))
    dz = None if z is None else dy * core * _dsilu(z)
    dc = dy if z is None else dy * _silu(z)
    # the adjoint g_t = C_t dc_t + a_{t+1} g_{t+1}, from the back
    g = dc[..., None] * Cm
    g[:, -1] += s["dstate"]
    nxt = torch.cat([a[:, 1:], torch.ones_like(a[:, :1])], 1)
    g = _prefix(nxt.flip(1), g.flip(1)).flip(1)
    B_, T, G, N = s["B"].shape
    sum_group = lambda t: t.unflatten(2, (G, D // G)).sum(3)  # noqa: E731
    dC = sum_group(dc[..., None] * h)
    dB = sum_group(g * (st * x)[..., None])
    first = torch.zeros_like(last) if s["state"] is None else s["state"]
    flow = g * a * torch.cat([first[:, None], h[:, :-1]], 1)
    gB = (g * Bm).sum(-1)
    dx = st * gB + s["D"] * dc
    dst = (flow * A).sum(-1) + gB * x
    draw_ = dst * torch.sigmoid(raw)
    if ok is not None:
        draw_ = torch.where(ok, draw_, torch.zeros_like(draw_))
    return dict(y=y.to(dt), state=last, dx=dx.to(dt), ddt=draw_.to(dt), dA=(flow * st[..., None]).sum((0, 1)), dB=dB.to(dt), dC=dC.to(dt),
                dD=(dc * x).sum((0, 1)), ddt_bias=draw_.sum((0, 1)),
                **_named(dz=None if z is None else dz.to(dt), dstate=None if s["state"] is None else a[:, 0] * g[:, 0]))


def _plain_scan_step(s):
    x, st = _f(s["x"]), _softplus(_f(s["dt"]) + s["dt_bias"])
    D = x.shape[-1]
    h = torch.exp(st[..., None] * s["A"]) * s["state"] + (st * x)[..., None] * _groups(_f(s["B"]), D)
    y = (h * _groups(_f(s["C"]), D)).sum(-1) + s["D"] * x
    if s["z"] is not None:
        y = y * _silu(_f(s["z"]))
    s["state"].copy_(h)
    return dict(y=y.to(s["x"].dtype), state=s["state"])


def _act(p, name):
    return p if name == "none" else _silu(p) if name == "silu" else 0.5 * p * (1 + torch.erf(p * math.sqrt(0.5)))


def _dact(p, name):
    if name == "none":
        return torch.ones_like(p)
    if name == "silu":
        return _dsilu(p)
    return 0.5 * (1 + torch.erf(p * math.sqrt(0.5))) + p * torch.exp(-0.5 * p * p) / math.sqrt(2 * math.pi)


def _plain_linear(s):
    x, w, act, dt = _f(s["x"]), _f(s["weight"]), s["case"]["act"], s["x"].dtype
    pre = x @ w.t()
    if s["bias"] is not None:
        pre = pre + _f(s["bias"])
    y = _act(pre, act)
    if s["residual"] is not None:
        y = y + _f(s["residual"])
    if not s["case"]["train"]:
        return dict(y=y.to(dt))
    dy = _f(s["dy"])
    dp = dy * _dact(pre, act)
    return dict(y=y.to(dt), dx=(dp @ w).to(dt), dweight=(dp.t() @ x).to(dt), **_named(
        dbias=None if s["bias"] is None else dp.sum(0).to(dt), dresidual=None if s["residual"] is None else s["dy"]))


_PLAIN = dict(conv=_plain_conv, conv_step=_plain_conv_step, scan=_plain_scan, scan_step=_plain_scan_step, linear=_plain_linear)


# ---- what a pass cannot do without ------------------------------------------------------------


def work(case):
    """Each input read once and each output written once; the formulas' operations, an exponential counted as one."""
    c = case
    if c["op"] == "linear":
        mnk, w = c["M"] * c["N"] * c["K"], 2
        n = c["M"] * c["K"] + c["N"] * c["K"] + c["M"] * c["N"] * (2 if c["residual"] else 1) + (c["N"] if c["bias"] else 0)
        if c["train"]:
            n += c["M"] * c["N"] + c["M"] * c["K"] + c["N"] * c["K"] + (c["N"] if c["bias"] else 0)
        return {"bytes": w * n, "flops": (6 if c["train"] else 2) * mnk}
    w = 2 if c["dtype"] == "bf16" else 4
    if c["op"] in ("conv", "conv_step"):
        B, T, C, W = c["B"], c.get("T", 1), c["C"], c["W"]
        own_size = C * W + (C if c["bias"] else 0)
        given = B * C * (W - 1) if c.get("state", True) else 0
        if c.get("train"):  # x, y, dy, dx; the weights and their gradients; the given state and its gradient
            n = 4 * B * T * C + 2 * own_size + 2 * given
        else:
            n = 2 * B * T * C + own_size + given + B * C * (W - 1)
        return {"bytes": w * n, "flops": B * T * C * (2 * W + 4) * (3 if c.get("train") else 1)}
    B, T, D, N, G = c["B"], c.get("T", 1), c["D"], c["N"], c["G"]
    tok = B * T * (3 * D + (D if c["gate"] else 0) + 2 * G * N)  # x, dt, z, B, C and y
    state = B * D * N * (2 if c["op"] == "scan_step" or c.get("state") else 1)
    n, flops = w * tok + 4 * (state + D * N + 2 * D), B * T * D * (7 * N + 10)
    if c.get("train"):  # dy, dx, ddt, dz, dB and dC are as many values again; the final state's gradient, the parameters'
        n += w * tok + 4 * (state + D * N + 2 * D)
        flops *= 4
    return {"bytes": n, "flops": flops}


# ---- the definitions in 64 bits ---------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    s = {k: v.double() if isinstance(v, torch.Tensor) and v.is_floating_point() else v for k, v in s.items()}
    return dict(conv=_exact_conv, conv_step=_exact_conv_step, scan=_exact_scan, scan_step=_exact_scan_step, linear=_exact_linear)[case["op"]](s)


def _with_grads(s, names, forward, outs):
    """``forward``'s outputs and, for a training case, its gradients by automatic differentiation."""
    names = [k for k in names if s[k] is not None]
    for k in names:
        s[k] = s[k].clone().requires_grad_()
    r = forward(s)
    grads = torch.autograd.grad([r[k] for k, _ in outs], [s[k] for k in names], [d for _, d in outs])
    return dict({k: v.detach() for k, v in r.items()}, **{"d" + k: g for k, g in zip(names, grads)})


def _exact_conv(s):
    c, F = s["case"], torch.nn.functional

    def forward(s):
        B, T, C = s["x"].shape
        W = s["weight"].shape[1]
        past = s["x"].new_zeros(B, C, W - 1) if s["state"] is None else s["state"]
        xp = torch.cat([past.transpose(1, 2), s["x"]], 1)
        y = sum(xp[:, w:w + T] * s["weight"][:, w] for w in range(W))
        y = y if s["bias"] is None else y + s["bias"]
        y = F.silu(y) if s["activation"] else y
        if s["lengths"] is not None:
            y = y * (torch.arange(T, device=y.device)[None, :, None] < s["lengths"][:, None, None])
        if c["train"]:
            return dict(y=y)
        ends = [T] * B if s["lengths"] is None else s["lengths"].tolist()
        return dict(y=y, state=torch.stack([xp[b, n:n + W - 1].t() for b, n in enumerate(ends)]))

    return _with_grads(s, ("x", "weight", "bias", "state"), forward, [("y", s["dy"])]) if c["train"] else forward(s)


def _exact_conv_step(s):
    xp = torch.cat([s["state"], s["x"][:, :, None]], 2)
    y = torch.einsum("bcw,cw->bc", xp, s["weight"])
    y = y if s["bias"] is None else y + s["bias"]
    return dict(y=torch.nn.functional.silu(y) if s["activation"] else y, state=xp[:, :, 1:])


def _exact_token(s, h, x, raw, Bt, Ct):
    """One token of the recurrence: (h, y before the gate, step size, decay), Bt and Ct (B, G, N)."""
    B, D = x.shape
    G = Bt.shape[1]
    st = torch.nn.functional.softplus(raw + s["dt_bias"], threshold=50.0)
    decay = torch.exp(st[:, :, None] * s["A"])
    rows = lambda t: t[:, :, None].expand(B, G, D // G, -1).reshape(B, D, -1)  # noqa: E731
    h = decay * h + (st * x)[:, :, None] * rows(Bt)
    return h, (h * rows(Ct)).sum(-1) + s["D"] * x, st, decay


def _exact_scan(s):
    c = s["case"]
    B, T, D = s["x"].shape
    G, N = s["B"].shape[2:]
    if B * T * D * N * (2 if c["train"] else 1) > 2**31:
        return None
    F = torch.nn.functional
    h = s["x"].new_zeros(B, D, N) if s["state"] is None else s["state"]
    live = [torch.ones(B, 1, device=h.device, dtype=torch.bool)] * T if s["lengths"] is None else \
        list((torch.arange(T, device=h.device)[:, None, None] < s["lengths"][:, None]).unbind(0))
    y, hs = torch.zeros_like(s["x"]), []
    for t in range(T):
        new, core, _, _ = _exact_token(s, h, s["x"][:, t], s["dt"][:, t], s["B"][:, t], s["C"][:, t])
        if c["train"]:
            hs.append(h)
        on = live[t].reshape(B, 1)
        h = torch.where(on[:, :, None], new, h) if s["lengths"] is not None else new
        y[:, t] = core * on if s["z"] is None else core * F.silu(s["z"][:, t]) * on
    if not c["train"]:
        return dict(y=y, state=h)
    # back through the tokens, each one's gradients by the product rule on the recurrence
    names = [k for k in ("x", "dt", "A", "B", "C", "D", "z", "dt_bias", "state") if s[k] is not None]
    grad = {k: torch.zeros(s[k].shape, device=h.device, dtype=torch.float64) for k in names}
    rows = lambda t: t[:, :, None].expand(B, G, D // G, -1).reshape(B, D, -1)  # noqa: E731
    g = s["dstate"]
    for t in range(T - 1, -1, -1):
        x, on = s["x"][:, t], live[t].reshape(B, 1).double()
        new, core, st, decay = _exact_token(s, hs[t], x, s["dt"][:, t], s["B"][:, t], s["C"][:, t])
        dy = s["dy"][:, t] * on
        if s["z"] is not None:
            zt = s["z"][:, t]
            sg = torch.sigmoid(zt)
            grad["z"][:, t] = dy * core * (sg + zt * sg * (1 - sg))
            dy = dy * zt * sg
        Bt, Ct = rows(s["B"][:, t]), rows(s["C"][:, t])
        gt = g * on[:, :, None] + dy[:, :, None] * Ct  # the adjoint of this token's state, where it is one
        per_group = lambda v: v.reshape(B, G, D // G, N).sum(2)  # noqa: E731
        grad["C"][:, t] = per_group(dy[:, :, None] * new)
        grad["B"][:, t] = per_group(gt * (st * x)[:, :, None])
        gb = (gt * Bt).sum(-1)
        grad["x"][:, t] = st * gb + s["D"] * dy
        fl = gt * decay * hs[t]
        dst = (fl * s["A"]).sum(-1) + gb * x
        dr = dst * torch.sigmoid(s["dt"][:, t] + s["dt_bias"])
        grad["dt"][:, t] = dr
        grad["dt_bias"] += dr.sum(0)
        grad["A"] += (fl * st[:, :, None]).sum(0)
        grad["D"] += (dy * x).sum(0)
        g = torch.where(on[:, :, None] > 0, gt * decay, g)
    if "state" in grad:
        grad["state"] = g
    return dict(y=y, state=h, **{"d" + k: v for k, v in grad.items()})


def _exact_scan_step(s):
    h, core, _, _ = _exact_token(s, s["state"], s["x"], s["dt"], s["B"], s["C"])
    return dict(y=core if s["z"] is None else core * torch.nn.functional.silu(s["z"]), state=h)


def _exact_linear(s):
    F, act = torch.nn.functional, s["case"]["act"]

    def forward(s):
        p = F.linear(s["x"], s["weight"], s["bias"])
        y = p if act == "none" else F.silu(p) if act == "silu" else F.gelu(p)
        return dict(y=y if s["residual"] is None else y + s["residual"])

    return _with_grads(s, ("x", "weight", "bias", "residual"), forward, [("y", s["dy"])]) if s["case"]["train"] else forward(s)
