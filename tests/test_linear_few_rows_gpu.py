"""ops.linear on both sides of the choice between its kernel for few rows and its tiles: up to 16, 32 and 64 rows, widths
and contractions below and above the bounds, aligned and not."""

import pytest
import torch

import ssm_reference as R
from archbench_b200 import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("odd", [False, True])
@pytest.mark.parametrize("N,K", [(2048, 512), (2056, 512), (4096, 264), (4104, 264), (16384, 72), (16392, 72), (64, 2816), (64, 2824),
                                 (96, 2048), (2048, 64), (40, 5000), (61, 513)])
@pytest.mark.parametrize("M", [1, 16, 17, 32, 33, 64])
def test_both_sides_of_the_choice(M, N, K, odd):
    g = torch.Generator("cuda").manual_seed(M + N + K)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda").bfloat16()
    pad = 3 if odd else 0
    off = lambda t: torch.nn.functional.pad(t, (pad, 2 * pad))[:, pad:pad + t.shape[1]]
    x, w, b, r = off(rnd(M, K)), off((rnd(N, K).float() / K ** 0.5).bfloat16()), rnd(N), off(rnd(M, N))
    y = ops.linear(x, w, b, "silu", r).double()
    want = R.linear(x.double(), w.double(), b.double(), "silu", r.double())
    # half a bf16 unit of the result, and fp32 sums of up to 5000 terms of rms 1 / sqrt(K): 2^-18 of 4 sigma
    assert ((y - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -16).all(), ((y - want).abs() - 2.0 ** -8 * want.abs()).max().item()
    assert ops.device_status() == 0
