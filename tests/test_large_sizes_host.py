"""Which sizes the C entry points take, without a GPU: past every check of sizes they only miss the device."""

import ctypes

import pytest

from archbench_b200 import ops, ssm_ops as S


def scan(B, T, D, N=16):
    return S.ScanArgs(x=0x1000, dt=0x2000, Bm=0x3000, Cm=0x4000, A=0x5000, y=0x6000, h_out=0x7000, sx_b=T * D, sx_t=D, sdt_b=T * D, sdt_t=D,
                      sB_b=T * N, sB_t=N, sB_g=N, sC_b=T * N, sC_t=N, sC_g=N, sy_b=T * D, sy_t=D, B=B, T=T, D=D, N=N, G=1, dtype=1)


@pytest.mark.parametrize("B,T,D,status", [(65535, 4, 64, -6), (65536, 4, 64, -6), (1 << 30, 4, 64, -6), ((1 << 30) + 1, 4, 64, -2),
                                          (1 << 18, 1 << 15, 64, -6), (1 << 20, 1 << 20, 128, -2), (2, (1 << 29) + 1, 8, -2)])
def test_scan_rows(B, T, D, status):
    lib, n = ops.load_library(), ctypes.c_size_t(0)
    a = scan(B, T, D)
    assert lib.gdn_scan_workspace_bytes(ctypes.byref(a), ctypes.byref(n)) == (0 if status == -6 else status)
    assert lib.gdn_scan_fwd(ctypes.byref(a), None) == status
    if status == -6:
        assert lib.gdn_scan_step(ctypes.byref(a), None) == status
    b = S.ScanBwdArgs(fwd=a, dy=0x8000, sdy_b=T * D, sdy_t=D, dx=0x9000, ddt=0xa000, dB=0xb000, dC=0xc000, dA=0xd000)
    b.fwd.ckpt = 0xe000
    assert lib.gdn_scan_bwd_workspace_bytes(ctypes.byref(b), ctypes.byref(n)) == (0 if status == -6 else status)
    b.fwd.workspace, b.fwd.workspace_bytes = 0x100000, n.value
    assert lib.gdn_scan_bwd(ctypes.byref(b), None) == status
