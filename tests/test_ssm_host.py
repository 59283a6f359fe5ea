"""Host side of the selective-state-space operators, without a GPU: argument blocks, the entry points' own refusals and
workspace sizes, module parameters, the registry and cache binding."""

import ctypes

import pytest
import torch
import torch.nn as nn

from archbench_b200 import linear_ops as L, ops, registry, ssm_ops as S
from archbench_b200.decode import bind_caches
from archbench_b200.lm import LM
from archbench_b200.ssm_layer import FusedMLP, SelectiveSSM


def lib():
    return ops.load_library()


def test_block_layouts():
    assert ctypes.sizeof(S.ConvArgs) == 7 * 8 + 7 * 8 + 4 * 4
    assert ctypes.sizeof(S.ConvBwdArgs) == ctypes.sizeof(S.ConvArgs) + 3 * 8 + 6 * 8 + 8
    assert ctypes.sizeof(S.ScanArgs) == 13 * 8 + 19 * 8 + 2 * 4 + 2 * 8
    assert ctypes.sizeof(S.ScanBwdArgs) == ctypes.sizeof(S.ScanArgs) + 3 * 8 + 10 * 8
    assert ctypes.sizeof(L.LinearArgs) == 6 * 8 + 7 * 8 + 2 * 4 + 2 * 8
    assert ctypes.sizeof(L.LinearBwdArgs) == 7 * 8 + 6 * 8 + 2 * 4 + 2 * 8
    assert all(hasattr(S.extension(), f) for f in ("causal_conv", "causal_conv_step", "selective_scan", "selective_scan_step", "linear"))


def conv(**kw):
    a = dict(x=0x1000, weight=0x2000, y=0x3000, sx_b=80, sx_t=8, sy_b=80, sy_t=8, B=2, T=10, C=8, width=4, act=1, dtype=1, w_dtype=1)
    return S.ConvArgs(**{**a, **kw})


def scan(**kw):
    a = dict(x=0x1000, dt=0x2000, Bm=0x3000, Cm=0x4000, A=0x5000, y=0x6000, sx_b=640, sx_t=64, sdt_b=640, sdt_t=64, sB_b=160, sB_t=16,
             sB_g=16, sC_b=160, sC_t=16, sC_g=16, sy_b=640, sy_t=64, B=2, T=10, D=64, N=16, G=1, dtype=1)
    return S.ScanArgs(**{**a, **kw})


def linear(**kw):
    a = dict(x=0x1000, weight=0x2000, y=0x3000, sx=64, sw=64, sy=32, M=100, N=32, K=64)
    return L.LinearArgs(**{**a, **kw})


@pytest.mark.parametrize("kw,status", [(dict(width=5), -5), (dict(width=1), -5), (dict(act=2), -5), (dict(dtype=7), -3), (dict(w_dtype=2), -3),
                                       (dict(weight=None), -1), (dict(x=None), -1), (dict(C=0), -2), (dict(B=-1), -2), (dict(sx_t=-8), -2)])
def test_conv_refusals(kw, status):
    assert lib().gdn_conv_fwd(ctypes.byref(conv(**kw)), None) == status


@pytest.mark.parametrize("kw,status", [(dict(N=65), -5), (dict(N=0), -2), (dict(G=3), -2), (dict(D=0), -2), (dict(dtype=2), -3), (dict(A=None), -1),
                                       (dict(Bm=None), -1), (dict(y=None), -1), (dict(T=-1), -2), (dict(sB_t=-1), -2)])
def test_scan_refusals(kw, status):
    assert lib().gdn_scan_fwd(ctypes.byref(scan(**kw)), None) == status


@pytest.mark.parametrize("kw,status", [(dict(N=0), -2), (dict(K=0), -2), (dict(M=-1), -2), (dict(act=3), -5), (dict(x=None), -1), (dict(y=None), -1),
                                       (dict(sx=-1), -2)])
def test_linear_refusals(kw, status):
    assert lib().gdn_linear_fwd(ctypes.byref(linear(**kw)), None) == status


def test_null_blocks_and_missing_workspaces():
    n = ctypes.c_size_t(0)
    for f in ("gdn_conv_fwd", "gdn_conv_step", "gdn_conv_bwd", "gdn_scan_fwd", "gdn_scan_step", "gdn_scan_bwd", "gdn_linear_fwd", "gdn_linear_bwd"):
        assert getattr(lib(), f)(None, None) == -1, f
    # a long row is split over time, an unaligned one is laid out again: both ask for scratch and refuse to run without
    for a in (scan(B=1, T=5000), scan(x=0x1002)):
        assert lib().gdn_scan_workspace_bytes(ctypes.byref(a), ctypes.byref(n)) == 0 and n.value > 0
        assert lib().gdn_scan_fwd(ctypes.byref(a), None) == -9
    assert lib().gdn_scan_workspace_bytes(ctypes.byref(scan()), ctypes.byref(n)) == 0 and n.value == 0
    a = linear(sx=63, K=63)
    assert lib().gdn_linear_workspace_bytes(ctypes.byref(a), ctypes.byref(n)) == 0 and n.value >= 100 * 64 * 2
    assert lib().gdn_linear_fwd(ctypes.byref(a), None) == -9
    b = S.ScanBwdArgs(fwd=scan(ckpt=0x7000), dy=0x8000, sdy_b=640, sdy_t=64, dx=0x9000, ddt=0xa000, dB=0xb000, dC=0xc000, dA=0xd000)
    assert lib().gdn_scan_bwd(ctypes.byref(b), None) == -9
    b.dA = None
    assert lib().gdn_scan_bwd(ctypes.byref(b), None) == -1


def test_offsets_past_32_bits_are_sized():
    n = ctypes.c_size_t(0)
    b = S.ScanBwdArgs(fwd=scan(B=64, T=100000, D=4096, sx_t=4096, sx_b=409600000))
    assert lib().gdn_scan_bwd_workspace_bytes(ctypes.byref(b), ctypes.byref(n)) == 0 and n.value > 2 ** 33


def test_convolution_sizes_past_64_bits_are_refused():
    assert lib().gdn_conv_fwd(ctypes.byref(conv(B=1 << 20, T=1 << 20, C=1 << 20)), None) == -2
    n = ctypes.c_size_t(0)
    b = S.ConvBwdArgs(fwd=conv(B=1 << 20, T=1 << 20, C=1 << 20))
    assert lib().gdn_conv_bwd_workspace_bytes(ctypes.byref(b), ctypes.byref(n)) == -2


def test_cpu_tensors_are_refused():
    x = torch.zeros(2, 3, 8)
    with pytest.raises(ValueError, match="CUDA"):
        ops.causal_conv(x, torch.zeros(8, 4))
    with pytest.raises(ValueError, match="CUDA"):
        ops.selective_scan(x, x, -torch.ones(8, 4), torch.zeros(2, 3, 4), torch.zeros(2, 3, 4))
    with pytest.raises(ValueError, match="CUDA"):
        ops.linear(x.bfloat16(), torch.zeros(4, 8).bfloat16())


def test_module_parameters():
    m = SelectiveSSM(48, state_size=8, expand=2)
    shapes = {k: tuple(v.shape) for k, v in m.state_dict().items()}
    assert shapes == {"in_proj.weight": (192, 48), "conv1d.weight": (96, 1, 4), "conv1d.bias": (96,), "x_proj.weight": (19, 96),
                      "dt_proj.weight": (96, 3), "dt_proj.bias": (96,), "A_log": (96, 8), "D": (96,), "out_proj.weight": (48, 96)}
    step = torch.nn.functional.softplus(m.dt_proj.bias)
    assert step.min() >= 0.99e-3 and step.max() <= 1.01e-1
    for bad in (dict(state_size=65), dict(conv_size=5)):
        with pytest.raises(ValueError):
            SelectiveSSM(48, **bad)
    with pytest.raises(ValueError):
        FusedMLP(48, 4.0, "relu")


def test_registry_lm_and_cache_binding():
    assert isinstance(registry.build_mixer("ssm", 64, 0, 2, state_size=8), SelectiveSSM)
    m = LM(arch="ssm", d_model=64, n_layer=2, vocab_size=32, mlp="silu", mlp_ratio=2.0)
    assert all(isinstance(b.mlp, FusedMLP) for b in m.blocks)
    with bind_caches(m) as caches:
        assert len(caches) == 2 and m.blocks[1].mixer.bound_cache is caches[1]
    assert m.blocks[1].mixer.bound_cache is None
    m.blocks[0].mixer = nn.Linear(64, 64)
    with pytest.raises(ValueError, match="no recurrent state"):
        with bind_caches(m):
            pass
