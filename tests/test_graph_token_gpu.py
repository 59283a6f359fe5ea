"""The captured decode step starts from the token it is given: a model whose greedy continuation changes from token to
token decodes the same ids replayed as eagerly."""

import pytest
import torch

from archbench_b200.decode import greedy_decode
from archbench_b200.lm import LM

pytestmark = pytest.mark.gpu


def test_graph_decode_follows_changing_tokens():
    torch.manual_seed(41)
    m = LM(arch="gdn", d_model=256, n_layer=2, vocab_size=512, layer=dict(num_heads=2, head_dim=128, expand_v=1.0), init_std=0.15).cuda().eval()
    # untied head: the next token is not the current one
    m.lm_head.weight = torch.nn.Parameter(torch.randn(512, 256, device="cuda"))
    idx = torch.randint(0, 512, (3, 70), device="cuda", generator=torch.Generator(device="cuda").manual_seed(42))
    ids_e = greedy_decode(m, idx, 12)
    assert (ids_e[:, 71:] != ids_e[:, 70:-1]).float().mean() > 0.5  # the premise
    assert torch.equal(ids_e, greedy_decode(m, idx, 12, graph=True))
