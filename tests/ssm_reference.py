"""Plain 64-bit forms of the selective-state-space operators and the fused linear layer, token by token, for the tests.
Differentiable by autograd."""

import torch
import torch.nn.functional as F


def conv(x, weight, bias=None, silu=False, state=None, lengths=None):
    B, T, C = x.shape
    W = weight.shape[1]
    past = x.new_zeros(B, C, W - 1) if state is None else state
    xp = torch.cat([past.transpose(1, 2), x], 1)
    y = sum(xp[:, w:w + T] * weight[:, w] for w in range(W))
    if bias is not None:
        y = y + bias
    if silu:
        y = F.silu(y)
    ends = [T] * B if lengths is None else [min(max(int(n), 0), T) for n in lengths]
    rows = [torch.cat([y[b, :n], torch.zeros_like(y[b, n:])]) for b, n in enumerate(ends)]
    last = torch.stack([xp[b, n:n + W - 1].t() for b, n in enumerate(ends)])
    return torch.stack(rows), last


def scan(x, dt, A, B, C, D=None, z=None, dt_bias=None, softplus=False, state=None, lengths=None):
    """B, C: (batch, T, G, N)."""
    b, T, Dm = x.shape
    G, N = B.shape[2:]
    h = x.new_zeros(b, Dm, N) if state is None else state
    ends = torch.full((b,), T) if lengths is None else lengths.clamp(0, T).cpu()
    rows = lambda t: t.repeat_interleave(Dm // G, dim=1)
    out = []
    for t in range(T):
        s = dt[:, t] if dt_bias is None else dt[:, t] + dt_bias
        if softplus:
            s = torch.logaddexp(s, torch.zeros_like(s))
        new = torch.exp(s[..., None] * A) * h + (s * x[:, t])[..., None] * rows(B[:, t])
        y = (new * rows(C[:, t])).sum(-1)
        if D is not None:
            y = y + D * x[:, t]
        if z is not None:
            y = y * F.silu(z[:, t])
        on = (t < ends).to(x.device)
        out.append(torch.where(on[:, None], y, torch.zeros_like(y)))
        h = torch.where(on[:, None, None], new, h)
    return (torch.stack(out, 1) if out else torch.zeros_like(x)), h


def linear(x, weight, bias=None, act=None, residual=None):
    p = F.linear(x, weight, bias)
    y = p if act is None else F.silu(p) if act == "silu" else F.gelu(p)
    return y if residual is None else y + residual


def close(got, want, what, accumulated=64):
    """|got - want| <= the rounding of the output's type (half a unit in the last place: 2^-9 of the value in bf16) plus
    `accumulated` fp32 roundings (2^-24 each) of the result's largest value -- the intermediate sums are of that size."""
    assert got.shape == want.shape, (what, got.shape, want.shape)
    if not want.numel():
        return
    g, w = got.detach().double().cpu(), want.detach().double().cpu()
    assert torch.isfinite(g).all(), what
    own = 2.0 ** -8 if got.dtype == torch.bfloat16 else 2.0 ** -23
    bound = own * w.abs() + accumulated * 2.0 ** -24 * w.abs().max() + 1e-30
    worst = ((g - w).abs() / bound).max().item()
    assert worst <= 1.0, f"{what}: {worst:.3g} times the bound"
