"""Projections that a user replaces, parametrises or hooks take part in the mixer's and the MLP's forward."""

import copy

import pytest
import torch
import torch.nn as nn
from torch.nn.utils import parametrize

from archbench_b200.layers import GDNCache
from archbench_b200.ssm_layer import FusedMLP, SelectiveSSM

pytestmark = pytest.mark.gpu


class Adapted(nn.Module):
    """A linear layer with a low-rank addition, as adapters make them: it keeps the layer it wraps."""

    def __init__(self, base):
        super().__init__()
        self.base = base
        self.down = nn.Linear(base.in_features, 2, bias=False)
        self.up = nn.Linear(2, base.out_features, bias=False)

    @property
    def weight(self):
        return self.base.weight

    @property
    def bias(self):
        return self.base.bias

    def forward(self, x):
        return self.base(x) + self.up(self.down(x))

    def merged(self):
        m = copy.deepcopy(self.base)
        with torch.no_grad():
            m.weight += self.up.weight @ self.down.weight
        return m


class Doubled(nn.Module):
    def forward(self, w):
        return 2 * w


LAYERS = {"ssm": (lambda: SelectiveSSM(64, bias=True), ("in_proj", "x_proj", "dt_proj", "out_proj")),
          "mlp": (lambda: FusedMLP(64, 2.0, "gelu"), ("up", "down"))}


def rnd(seed, *s):
    return torch.randn(*s, generator=torch.Generator("cuda").manual_seed(seed), device="cuda")


@pytest.mark.parametrize("kind", LAYERS)
def test_replaced_and_parametrised_projections(kind):
    make, names = LAYERS[kind]
    x, r = rnd(1, 2, 6, 64), rnd(2, 2, 6, 64)
    for name in names:
        torch.manual_seed(3)
        m = make().cuda()
        merged, doubled = copy.deepcopy(m), copy.deepcopy(m)
        ad = Adapted(getattr(m, name)).cuda()
        setattr(m, name, ad)
        setattr(merged, name, ad.merged())
        with torch.no_grad():
            want, got = merged(x, residual=r), m(x, residual=r)
            assert ((got - want).norm() <= 1e-5 * want.norm()).item(), name  # fp32: the same sums in another order
            other = copy.deepcopy(doubled)
            parametrize.register_parametrization(getattr(doubled, name), "weight", Doubled())
            getattr(other, name).weight.mul_(2)
            a, b = doubled(x, residual=r), other(x, residual=r)
            assert ((a - b).norm() <= 1e-5 * b.norm()).item(), name


@pytest.mark.parametrize("kind", LAYERS)
def test_hooks_run(kind):
    make, names = LAYERS[kind]
    torch.manual_seed(4)
    m = make().cuda().bfloat16()
    x, r = rnd(5, 2, 6, 64).bfloat16(), rnd(6, 2, 6, 64).bfloat16()
    with torch.no_grad():
        want = m(x, residual=r)
    seen = []
    for name in names:
        getattr(m, name).register_forward_hook(lambda mod, a, out, name=name: seen.append((name, tuple(out.shape))))
    with torch.no_grad():
        got = m(x, residual=r)
    assert [n for n, _ in seen] == list(names)
    assert ((got - want).float().norm() <= 2e-2 * want.float().norm()).item()


def test_adapted_mixer_decodes_what_it_prefills():
    torch.manual_seed(7)
    m = SelectiveSSM(64).cuda()
    m.dt_proj, m.in_proj = Adapted(m.dt_proj).cuda(), Adapted(m.in_proj).cuda()
    x = rnd(8, 3, 9, 64)
    with torch.no_grad():
        want, cache = m(x), GDNCache()
        got = torch.cat([m(x[:, :5], cache)] + [m(x[:, t:t + 1], cache) for t in range(5, 9)], 1)
    assert ((got - want).norm() <= 1e-5 * want.norm()).item()


class Scaled(nn.Module):
    """A convolution that is more than its weight."""

    def __init__(self, base):
        super().__init__()
        self.base = base

    weight = property(lambda self: self.base.weight)
    bias = property(lambda self: self.base.bias)

    def forward(self, x):
        return 2 * self.base(x)


@pytest.mark.parametrize("how", ["replaced", "hooked", "parametrised"])
def test_convolution_of_another_kind(how):
    torch.manual_seed(9)
    m = SelectiveSSM(64).cuda()
    want = copy.deepcopy(m)
    with torch.no_grad():
        want.conv1d.weight.mul_(2)
        if how != "parametrised":
            want.conv1d.bias.mul_(2)
    if how == "replaced":
        m.conv1d = Scaled(m.conv1d)
    elif how == "hooked":
        m.conv1d.register_forward_hook(lambda mod, args, out: 2 * out)
    else:
        parametrize.register_parametrization(m.conv1d, "weight", Doubled())
    x = rnd(10, 3, 9, 64)
    with torch.no_grad():
        a, b, cache = want(x), m(x), GDNCache()
        c = torch.cat([m(x[:, :1], cache), m(x[:, 1:5], cache)] + [m(x[:, t:t + 1], cache) for t in range(5, 9)], 1)
    for got in (b, c):
        assert ((got - a).norm() <= 1e-5 * a.norm()).item()
    ga = torch.autograd.grad(want(x).sum(), want.in_proj.weight)[0]
    gb = torch.autograd.grad(m(x).sum(), m.in_proj.weight)[0]
    assert ((ga - gb).norm() <= 1e-5 * ga.norm()).item()
