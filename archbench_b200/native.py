"""The native library ``libgdn_b200.so``: where it is, its symbols, its dtype codes and its errors.

Each operator module adds the entry points it calls to ``SYMBOLS``; ``load_library`` checks that the library has them
all."""

from __future__ import annotations

import ctypes
import os

import torch

_PKG = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_PKG, "libgdn_b200.so")

GDN_DTYPE_F32, GDN_DTYPE_BF16 = 0, 1
_DT = {torch.float32: GDN_DTYPE_F32, torch.bfloat16: GDN_DTYPE_BF16}

SYMBOLS: dict = {}  # name -> (argtypes, restype)

_LIB = None


class GdnError(RuntimeError):
    """A gdn_status error returned by the native library."""

    def __init__(self, status: int, msg: str):
        super().__init__(f"gdn_b200 error {status}: {msg}")
        self.status = status


def load_library(path: str = LIB_PATH):
    """Load libgdn_b200.so (built by ``python -m archbench_b200.build``); raises if absent."""
    global _LIB
    if _LIB is not None and path == LIB_PATH:
        return _LIB
    if not os.path.exists(path):
        raise FileNotFoundError(f"{path} is missing: build it with `python -m archbench_b200.build`")
    lib = ctypes.CDLL(path)
    for name, (argtypes, restype) in SYMBOLS.items():
        fn = getattr(lib, name)
        fn.argtypes = argtypes
        fn.restype = restype
    if path == LIB_PATH:
        _LIB = lib
    return lib


def _check(status: int):
    if status != 0:
        msg = load_library().gdn_status_string(status)
        raise GdnError(status, msg.decode() if msg else "?")


def _check_cuda(*ts):
    for t in ts:
        if t is not None and not t.is_cuda:
            raise ValueError("archbench_b200 ops run on CUDA tensors only (no CPU path)")
