"""Gradients around the one-token forms: the operators have none and say so, and the mixer takes the differentiable
forms where a gradient is wanted."""

import pytest
import torch

from archbench_b200 import ops
from archbench_b200.layers import GDNCache
from archbench_b200.ssm_layer import SelectiveSSM

pytestmark = pytest.mark.gpu


def rnd(g, *s):
    return torch.randn(*s, generator=g, device="cuda")


def test_one_token_outputs_refuse_to_be_differentiated():
    g = torch.Generator("cuda").manual_seed(1)
    x, w, A, B = rnd(g, 2, 8), rnd(g, 8, 4), -torch.ones(8, 4, device="cuda"), rnd(g, 2, 4)
    sc, ss = torch.zeros(2, 8, 3, device="cuda"), torch.zeros(2, 8, 4, device="cuda")
    for leaf in (x, w):
        leaf.requires_grad_()
        y = ops.causal_conv_step(x, w, sc, activation="silu")
        assert y.requires_grad
        with pytest.raises(RuntimeError, match="one-token"):
            y.sum().backward()
        leaf.requires_grad_(False)
    for leaf in (x, A, B):
        leaf.requires_grad_()
        y = ops.selective_scan_step(x, x, A, B, B, ss, dt_softplus=True)
        assert y.requires_grad
        with pytest.raises(RuntimeError, match="one-token"):
            y.sum().backward()
        leaf.requires_grad_(False)
    x.requires_grad_()
    with torch.no_grad():
        assert not ops.causal_conv_step(x, w, sc).requires_grad


def test_one_token_forms_refuse_a_state_with_history():
    g = torch.Generator("cuda").manual_seed(2)
    x, w, A, B = rnd(g, 2, 8), rnd(g, 8, 4), -torch.ones(8, 4, device="cuda"), rnd(g, 2, 4)
    sc, ss = torch.zeros(2, 8, 3, device="cuda", requires_grad=True), torch.zeros(2, 8, 4, device="cuda", requires_grad=True)
    for s in (sc, sc * 2):
        with pytest.raises(ValueError, match="detach"):
            ops.causal_conv_step(x, w, s)
    for s in (ss, ss * 2):
        with pytest.raises(ValueError, match="detach"):
            ops.selective_scan_step(x, x, A, B, B, s)
    with torch.no_grad():
        ops.causal_conv_step(x, w, sc)
        ops.selective_scan_step(x, x, A, B, B, ss)


def test_mixer_trains_through_a_cached_token():
    """The gradient of a call on one token that continues a cache: that of the same token inside one longer call."""
    torch.manual_seed(4)
    m = SelectiveSSM(64).cuda()
    x = rnd(torch.Generator("cuda").manual_seed(5), 2, 6, 64)
    dy = rnd(torch.Generator("cuda").manual_seed(6), 2, 1, 64)
    want = torch.autograd.grad((m(x)[:, 5:] * dy).sum(), list(m.parameters()))
    cache = GDNCache()
    m(x[:, :5], cache)
    y = m(x[:, 5:], cache)
    got = torch.autograd.grad((y * dy).sum(), list(m.parameters()))
    assert cache.seen == 6
    for (n, _), a, b in zip(m.named_parameters(), got, want):
        # the same fp32 sums in two pieces: 2^-24 per rounding, a few hundred of them
        assert ((a - b).norm() <= 1e-5 * b.norm() + 1e-9).item(), n


def test_captured_decoding_outside_no_grad():
    """A captured step never records history, whatever the caller's mode."""
    from archbench_b200.decode import GraphDecoder, bind_caches, greedy_decode
    from archbench_b200.lm import LM

    torch.manual_seed(7)
    m = LM(arch="ssm", d_model=128, n_layer=2, vocab_size=256, mlp_ratio=2.0, mlp="gelu", init_std=0.1).cuda().bfloat16()
    idx = torch.randint(0, 256, (3, 12), device="cuda", generator=torch.Generator("cuda").manual_seed(8))
    want = greedy_decode(m, idx, 6)
    with bind_caches(m) as caches:
        tokens = [m(idx)[0][:, -1].argmax(-1)]  # a prompt with history: the caches carry it
        dec = GraphDecoder(m, caches, tokens[0])
        for _ in range(5):
            dec.step()
            tokens.append(dec.token.clone())
    assert torch.equal(torch.stack(tokens, 1), want[:, 12:])
