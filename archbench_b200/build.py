"""Build the native library ``libgdn_b200.so`` in-tree with nvcc for sm_100a.

    python -m archbench_b200.build            # incremental
    python -m archbench_b200.build --force

Each ``csrc/*.cu`` compiles to an object under ``_build/`` and the objects link into
``archbench_b200/libgdn_b200.so`` (static CUDA runtime, C ABI of ``include/gdn_b200.h``).  ``csrc/torch_ops.cpp``, the
operators as functions of torch tensors, compiles with the host compiler to the extension module
``archbench_b200/_torch_ops.so``, which links against that library beside it.  Where the host compiler, ``Python.h`` or torch
is missing, the library is built without it.
"""

from __future__ import annotations

import concurrent.futures as cf
import importlib.metadata
import importlib.util
import os
import shlex
import shutil
import subprocess
import sys
import sysconfig

PKG = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG)
CSRC = os.path.join(PKG, "csrc")
OBJ = os.path.join(PKG, "_build")
LIB = os.path.join(PKG, "libgdn_b200.so")
TORCH_OPS = os.path.join(PKG, "_torch_ops.so")
INCLUDE = os.path.join(ROOT, "include")

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ["-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC,-O2", "--expt-relaxed-constexpr", "-Xptxas", "-v"]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise FileNotFoundError("nvcc not found")


def _sources():
    return sorted(os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith(".cu"))


def _headers():
    hs = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".cuh", ".h"))]
    hs += [os.path.join(INCLUDE, f) for f in os.listdir(INCLUDE) if f.endswith(".h")]
    return hs


def _compile(src, force, verbose):
    obj = os.path.join(OBJ, os.path.basename(src)[:-3] + ".o")
    newest_dep = max([os.path.getmtime(src)] + [os.path.getmtime(h) for h in _headers()])
    if not force and os.path.exists(obj) and os.path.getmtime(obj) >= newest_dep:
        return obj, ""
    cmd = [nvcc(), *ARCH, *NVCC_FLAGS, "-I", INCLUDE, "-I", CSRC, "-c", src, "-o", obj]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"nvcc failed on {src}:\n{r.stdout}\n{r.stderr}")
    return obj, r.stderr if verbose else ""


def _cxx():
    return shlex.split(os.environ.get("CXX", "g++"))


def _torch_ops_lack():
    """What the torch extension needs and this machine lacks, or None.  The library itself needs nvcc alone."""
    if shutil.which(_cxx()[0]) is None:
        return f"no host compiler {_cxx()[0]}"
    if not os.path.exists(os.path.join(sysconfig.get_paths()["include"], "Python.h")):
        return "no Python.h"
    if importlib.util.find_spec("torch") is None:
        return "no torch"
    return None


def _torch_ops_sources():
    return [os.path.join(CSRC, "torch_ops.cpp"), os.path.join(INCLUDE, "gdn_b200.h")]


def _torch_ops_built_for():
    """What the extension's binary interface hangs on beside its sources."""
    return f"torch {importlib.metadata.version('torch')}, python {sys.version}, {' '.join(_cxx())}\n"


def _compile_torch_ops(force):
    """The object of the torch extension (30 s with torch's headers)."""
    deps = _torch_ops_sources()
    src, obj = deps[0], os.path.join(OBJ, "torch_ops.o")
    built_for = os.path.join(OBJ, "torch_ops.txt")
    same = os.path.exists(built_for) and open(built_for).read() == _torch_ops_built_for()
    if not force and same and os.path.exists(obj) and os.path.getmtime(obj) >= max(os.path.getmtime(d) for d in deps):
        return obj
    import torch

    inc = os.path.join(os.path.dirname(torch.__file__), "include")
    cuda = os.path.join(os.path.dirname(os.path.dirname(nvcc())), "include")
    dirs = [inc, os.path.join(inc, "torch", "csrc", "api", "include"), cuda, sysconfig.get_paths()["include"]]
    cmd = [*_cxx(), "-O2", "-std=c++17", "-fPIC", "-c", src, "-o", obj, "-DTORCH_EXTENSION_NAME=_torch_ops",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", "-I", INCLUDE]
    for d in dirs:
        cmd += ["-isystem", d]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"{cmd[0]} failed on {src}:\n{r.stdout}\n{r.stderr}")
    with open(built_for, "w") as f:
        f.write(_torch_ops_built_for())
    return obj


def _link_torch_ops(obj, force):
    if not force and os.path.exists(TORCH_OPS) and os.path.getmtime(TORCH_OPS) >= os.path.getmtime(obj):
        return
    import torch

    lib = os.path.join(os.path.dirname(torch.__file__), "lib")
    tmp = TORCH_OPS + ".tmp"
    cmd = [*_cxx(), "-shared", "-o", tmp, obj, "-L" + lib, "-lc10", "-ltorch_cpu", "-ltorch", "-ltorch_python", "-lc10_cuda",
           "-L" + PKG, "-l:libgdn_b200.so", "-Wl,-rpath,$ORIGIN"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link of {TORCH_OPS} failed:\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, TORCH_OPS)


def build(force: bool = False, verbose: bool = False) -> str:
    os.makedirs(OBJ, exist_ok=True)
    srcs = _sources()
    with cf.ThreadPoolExecutor(max_workers=min(8, len(srcs)) + 1) as ex:
        lack = _torch_ops_lack()
        torch_obj = None if lack else ex.submit(_compile_torch_ops, force)
        results = list(ex.map(lambda s: _compile(s, force, verbose), srcs))
    objs = [o for o, _ in results]
    for _, log in results:
        if log:
            print(log, file=sys.stderr)
    if force or not os.path.exists(LIB) or os.path.getmtime(LIB) < max(os.path.getmtime(o) for o in objs):
        tmp = LIB + ".tmp"
        cmd = [nvcc(), *ARCH, "-shared", "-Xcompiler", "-fPIC", "-o", tmp, *objs]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
        os.replace(tmp, LIB)
    if lack:
        if os.path.exists(TORCH_OPS) and os.path.getmtime(TORCH_OPS) < max(os.path.getmtime(d) for d in _torch_ops_sources()):
            os.remove(TORCH_OPS)  # none rather than one of other sources: the operators that need it then name it
        print(f"{os.path.basename(TORCH_OPS)} not built: {lack}", file=sys.stderr)
    else:
        _link_torch_ops(torch_obj.result(), force)  # a failure here leaves the library built
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
