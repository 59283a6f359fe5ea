"""The selective-state-space mixer and the fused MLP under autocast: the residual stream keeps its type."""

import pytest
import torch

from archbench_b200.lm import LM, Block
from archbench_b200.ssm_layer import FusedMLP, SelectiveSSM

pytestmark = pytest.mark.gpu


def rnd(seed, *s):
    return torch.randn(*s, generator=torch.Generator("cuda").manual_seed(seed), device="cuda")


@pytest.mark.parametrize("part", [lambda: SelectiveSSM(64), lambda: FusedMLP(64, 2.0, "gelu")])
def test_residual_keeps_its_type(part):
    """bf16 work on an fp32 stream adds to it in fp32: nothing of the stream is rounded."""
    torch.manual_seed(1)
    m = part().cuda()
    x, r, dy = rnd(2, 3, 7, 64), (100 * rnd(3, 3, 7, 64)).requires_grad_(), rnd(4, 3, 7, 64)
    with torch.autocast("cuda", torch.bfloat16):
        y, alone = m(x, residual=r), m(x)
    assert y.dtype == torch.float32 and alone.dtype == torch.bfloat16
    assert torch.equal(y, alone.float() + r)
    assert torch.equal(torch.autograd.grad(y, r, dy)[0], dy)


def test_block_stream_under_autocast():
    """Four blocks on a stream of fp32: as near to the 64-bit stream as the parts' bf16 outputs allow.

    A part's output is off by a few bf16 roundings of itself (2^-9 rms each, ten along the chain: 1 % at most); the
    stream of size 100 would take 2^-9 of 100 per rounding."""
    torch.manual_seed(5)
    blocks = [Block("ssm", 64, i, 4, 2.0, 1e-5, {}, "gelu").cuda() for i in range(4)]
    x = 100 * rnd(6, 2, 9, 64)
    with torch.no_grad():
        h32, h = x.clone(), x.clone()
        for b in blocks:
            h32 = b(h32)  # fp32 all along: 1e-6 off at most
        with torch.autocast("cuda", torch.bfloat16):
            for b in blocks:
                h = b(h)
    assert h.dtype == torch.float32
    moved = (h32 - x).norm()
    assert ((h - h32).norm() <= 0.03 * moved).item(), ((h - h32).norm() / moved).item()


def test_lm_trains_under_autocast():
    torch.manual_seed(7)
    m = LM(arch="ssm", d_model=128, n_layer=2, vocab_size=256, mlp_ratio=2.0, mlp="silu", init_std=0.1).cuda()
    idx = torch.randint(0, 256, (4, 33), device="cuda", generator=torch.Generator("cuda").manual_seed(8))
    with torch.autocast("cuda", torch.bfloat16):
        _, loss = m(idx[:, :-1], idx[:, 1:])
    loss.backward()
    _, loss32 = m(idx[:, :-1], idx[:, 1:])
    assert abs(loss.item() - loss32.item()) <= 1e-2 * loss32.item()
    assert all(p.grad is not None and p.grad.dtype == torch.float32 and torch.isfinite(p.grad).all() for p in m.parameters())
