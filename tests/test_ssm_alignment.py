"""Buffers off the boundaries that vector accesses need, through the C entry points: refused where a workspace is (on the
host, without a GPU), served by narrower accesses elsewhere (on the GPU)."""

import ctypes

import pytest
import torch

import ssm_reference as R
from archbench_b200 import linear_ops as L, ops, ssm_ops as S


def scan(**kw):
    a = dict(x=0x1000, dt=0x2000, Bm=0x3000, Cm=0x4000, A=0x5000, y=0x6000, sx_b=320000, sx_t=64, sdt_b=320000, sdt_t=64, sB_b=80000, sB_t=16,
             sB_g=16, sC_b=80000, sC_t=16, sC_g=16, sy_b=320000, sy_t=64, B=1, T=5000, D=64, N=16, G=1, dtype=1)
    return S.ScanArgs(**{**a, **kw})


def status_and_size(query, call, block, set_workspace):
    """The entry point's status with a workspace of the size that it asks for, 8 bytes off a 16-byte boundary."""
    n = ctypes.c_size_t(0)
    lib = ops.load_library()
    assert getattr(lib, query)(ctypes.byref(block), ctypes.byref(n)) == 0 and n.value > 0
    set_workspace(block, 0x100008, n.value)
    return getattr(lib, call)(ctypes.byref(block), None)


def test_workspaces_off_their_boundary_are_refused():
    def own(b, p, n):
        b.workspace, b.workspace_bytes = p, n

    def inner(b, p, n):
        own(b.fwd, p, n)

    assert status_and_size("gdn_scan_workspace_bytes", "gdn_scan_fwd", scan(), own) == -4
    b = S.ScanBwdArgs(fwd=scan(ckpt=0x7000), dy=0x8000, sdy_b=320000, sdy_t=64, dx=0x9000, ddt=0xa000, dB=0xb000, dC=0xc000, dA=0xd000)
    assert status_and_size("gdn_scan_bwd_workspace_bytes", "gdn_scan_bwd", b, inner) == -4
    f = L.LinearArgs(x=0x1000, weight=0x2000, y=0x3000, sx=63, sw=63, sy=32, M=100, N=32, K=63)
    assert status_and_size("gdn_linear_workspace_bytes", "gdn_linear_fwd", f, own) == -4
    g = L.LinearBwdArgs(x=0x1000, weight=0x2000, pre=0x3000, dy=0x4000, dx=0x5000, dweight=0x6000, sx=64, sw=64, sdy=32, M=100, N=32, K=64, act=1)
    assert status_and_size("gdn_linear_bwd_workspace_bytes", "gdn_linear_bwd", g, own) == -4


class Arena:
    """Device tensors whose first value stands `off` values past a 256-byte boundary, with untouched values around."""

    GUARD = 64

    def __init__(self):
        self.made = []

    def __call__(self, shape, dtype, off, like=None):
        n = 1
        for s in shape:
            n *= s
        buf = torch.full((n + off + 2 * self.GUARD,), 77.0, device="cuda", dtype=dtype)
        t = buf[self.GUARD + off:self.GUARD + off + n].view(shape)
        if like is not None:
            t.copy_(like)
        self.made.append((buf, self.GUARD + off, n))
        return t

    def intact(self):
        return all((b[:a] == 77).all() and (b[a + n:] == 77).all() for b, a, n in self.made)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,T,D,N", [(2, 37, 24, 16), (1, 300, 20, 4), (2, 41, 22, 8), (1, 520, 16, 5)])
@pytest.mark.parametrize("off_ckpt,off_out,off_A", [(1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 1, 1), (2, 3, 0)])
def test_scan_buffers_anywhere(dtype, B, T, D, N, off_ckpt, off_out, off_A):
    """Checkpoints, gradients and A one to three values off: forward and backward as everywhere."""
    g = torch.Generator("cuda").manual_seed(T + D)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")
    at, f32 = Arena(), torch.float32
    x, dt, z, dy = (at((B, T, D), dtype, 0, rnd(B, T, D)) for _ in range(4))
    Bm, C = (at((B, T, 1, N), dtype, 0, rnd(B, T, 1, N)) for _ in range(2))
    A = at((D, N), f32, off_A, -torch.rand(D, N, generator=g, device="cuda") - 0.1)
    y, h = at((B, T, D), dtype, off_out), at((B, D, N), f32, off_A)
    ckpt = at((B, (T + 7) // 8, D, N), f32, off_ckpt)
    a = S.ScanArgs(x=x.data_ptr(), dt=dt.data_ptr(), Bm=Bm.data_ptr(), Cm=C.data_ptr(), z=z.data_ptr(), A=A.data_ptr(), y=y.data_ptr(),
                   h_out=h.data_ptr(), ckpt=ckpt.data_ptr(), B=B, T=T, D=D, N=N, G=1, dtype=0 if dtype == f32 else 1, softplus=1)
    for k, w in (("x", D), ("dt", D), ("z", D), ("y", D), ("B", N), ("C", N)):
        setattr(a, f"s{k}_b", T * w)
        setattr(a, f"s{k}_t", w)
    a.sB_g = a.sC_g = N
    lib, s, n = ops.load_library(), torch.cuda.current_stream().cuda_stream, ctypes.c_size_t(0)
    assert lib.gdn_scan_workspace_bytes(ctypes.byref(a), ctypes.byref(n)) == 0
    ws = torch.empty(n.value + 1, device="cuda", dtype=torch.uint8)
    a.workspace, a.workspace_bytes = ws.data_ptr(), n.value
    assert lib.gdn_scan_fwd(ctypes.byref(a), s) == 0
    dx, ddt, dz = (at((B, T, D), dtype, off_out) for _ in range(3))
    dB, dC = (at((B, T, 1, N), dtype, off_out) for _ in range(2))
    dA, dh0 = at((D, N), f32, off_out), at((B, D, N), f32, off_A)
    b = S.ScanBwdArgs(fwd=a, dy=dy.data_ptr(), sdy_b=T * D, sdy_t=D, dx=dx.data_ptr(), ddt=ddt.data_ptr(), dB=dB.data_ptr(), dC=dC.data_ptr(),
                      dz=dz.data_ptr(), dA=dA.data_ptr(), dh0=dh0.data_ptr())
    assert lib.gdn_scan_bwd_workspace_bytes(ctypes.byref(b), ctypes.byref(n)) == 0
    ws2 = torch.empty(n.value + 1, device="cuda", dtype=torch.uint8)
    b.fwd.workspace, b.fwd.workspace_bytes = ws2.data_ptr(), n.value
    assert lib.gdn_scan_bwd(ctypes.byref(b), s) == 0
    torch.cuda.synchronize()
    assert at.intact()
    ref = [t.double().cpu().requires_grad_() for t in (x, dt, A, Bm, C, z)]
    h0 = torch.zeros(B, D, N, dtype=torch.double, requires_grad=True)
    y0, last = R.scan(*ref[:5], z=ref[5], softplus=True, state=h0)
    R.close(y, y0, "y", accumulated=128 + N)
    R.close(h, last, "state", accumulated=128)
    want = torch.autograd.grad(y0, [*ref, h0], dy.double().cpu())
    for k, p, q in zip(("x", "dt", "A", "B", "C", "z", "h0"), (dx, ddt, dA, dB, dC, dz, dh0), want):
        R.close(p, q, "d" + k, accumulated=256 + (B * T if k == "A" else D if k in "BC" else 0))


@pytest.mark.gpu
@pytest.mark.parametrize("train", [False, True])
def test_scan_with_a_parameter_off_its_boundary(train):
    """The same by the package's own call: A a contiguous view one value into its storage."""
    g = torch.Generator("cuda").manual_seed(9)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")
    store = torch.zeros(24 * 16 + 1, device="cuda")
    store[1:] = -torch.rand(24 * 16, generator=g, device="cuda") - 0.1
    A = store[1:].view(24, 16)
    assert A.is_contiguous() and A.data_ptr() % 16
    v = [rnd(2, 530, 24), rnd(2, 530, 24), A, rnd(2, 530, 1, 16), rnd(2, 530, 1, 16)]
    own = [t.detach().requires_grad_(train) for t in v]
    ref = [t.double().cpu().requires_grad_() for t in v]
    y, h = ops.selective_scan(*own, dt_softplus=True, output_final_state=True)
    y0, h0 = R.scan(*ref, softplus=True)
    R.close(y, y0, "y", accumulated=128 + 16)
    R.close(h, h0, "state", accumulated=128)
    if train:
        dy = rnd(2, 530, 24)
        for k, p, q in zip(("x", "dt", "A", "B", "C"), torch.autograd.grad(y, own, dy), torch.autograd.grad(y0, ref, dy.double().cpu())):
            R.close(p, q, "d" + k, accumulated=256 + (2 * 530 if k == "A" else 24 if k in "BC" else 0))
