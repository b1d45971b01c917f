"""Build ``libgsplat_b200.so`` in-tree with nvcc for sm_100a.

Usage: ``python -m mlx_gsplat_b200.build`` (or ``build()`` from Python).
The library is a plain C ABI (``include/gsplat_b200.h``) loaded with ctypes;
no PyTorch headers are involved.  Beside it ``libgsplat_tensors.so``
(``csrc/tensors.cpp``, g++ with torch's headers) reads torch tensors' metadata
for the many-tensor calls; it holds no kernels, and where it cannot be compiled
the package does the same in Python.
"""
from __future__ import annotations

import glob
import os
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

PKG = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG)
CSRC = os.path.join(PKG, "csrc")
INCLUDE = os.path.join(ROOT, "include")
LIB = os.path.join(PKG, "libgsplat_b200.so")
TENSORS_SRC = os.path.join(CSRC, "tensors.cpp")
TENSORS_LIB = os.path.join(PKG, "libgsplat_tensors.so")
BUILD_DIR = os.path.join(PKG, "_build")

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC",
    "--expt-relaxed-constexpr", "-Xptxas", "-warn-spills",
]


def _nvcc() -> str:
    cand = os.environ.get("NVCC") or shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(cand):
        raise RuntimeError("nvcc not found; set NVCC")
    return cand


def sources():
    return sorted(glob.glob(os.path.join(CSRC, "*.cu")))


def build_tensors() -> str:
    """Compile the tensor helper against the installed torch."""
    import sysconfig

    import torch

    from . import _lib
    root = os.path.dirname(torch.__file__)
    includes = [os.path.join(root, "include"), os.path.join(root, "include", "torch", "csrc", "api", "include"),
                sysconfig.get_paths()["include"]]
    tmp = TENSORS_LIB + ".tmp"
    cmd = [os.environ.get("CXX") or shutil.which("g++") or "g++", "-O2", "-std=c++17", "-shared", "-fPIC",
           f'-DGST_ABI="{_lib.tensors_abi()}"',
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", *(f"-isystem{i}" for i in includes),
           "-I", INCLUDE, TENSORS_SRC, "-o", tmp, "-L" + os.path.join(root, "lib"), "-ltorch_python", "-ltorch_cpu",
           "-lc10"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError("g++ failed for tensors.cpp:\n" + r.stderr)
    os.replace(tmp, TENSORS_LIB)
    return TENSORS_LIB


def _older(lib, deps) -> bool:
    return not os.path.exists(lib) or any(os.path.getmtime(d) > os.path.getmtime(lib) for d in deps)


def _headers():
    return glob.glob(os.path.join(INCLUDE, "*.h"))


def _stale(objs, srcs) -> bool:
    return _older(LIB, srcs + glob.glob(os.path.join(CSRC, "*.cuh")) + _headers())


def _tensors_stale() -> bool:
    if _older(TENSORS_LIB, [TENSORS_SRC] + _headers()):
        return True
    from . import _lib
    try:
        _lib.load_tensors(TENSORS_LIB)
    except OSError:  # compiled against another torch
        return True
    return False


def _try_tensors() -> None:
    """Compiles the tensor helper; without it (no g++, no headers of torch or
    Python) the rest of the package works the same."""
    try:
        build_tensors()
    except (RuntimeError, OSError) as e:
        if os.path.exists(TENSORS_LIB):
            os.remove(TENSORS_LIB)  # of other sources or another torch
        print(f"the tensor helper was not built, tensors will be read in Python: {e}", file=sys.stderr)


def build(force: bool = False, verbose: bool = False, extra_flags=None) -> str:
    srcs = sources()
    os.makedirs(BUILD_DIR, exist_ok=True)
    objs = [os.path.join(BUILD_DIR, os.path.basename(s)[:-3] + ".o") for s in srcs]
    helper = force or _tensors_stale()
    if not force and not _stale(objs, srcs):
        if helper:
            _try_tensors()
        return LIB
    nvcc = _nvcc()
    flags = NVCC_FLAGS + list(extra_flags or [])

    def compile_one(pair):
        src, obj = pair
        cmd = [nvcc, *flags, "-I", INCLUDE, "-I", CSRC, "-c", src, "-o", obj]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"nvcc failed for {os.path.basename(src)}:\n{r.stderr}")
        return r.stderr

    with ThreadPoolExecutor(max_workers=min(8, len(srcs))) as ex:
        tensors = ex.submit(_try_tensors) if helper else None
        logs = list(ex.map(compile_one, zip(srcs, objs)))
        if tensors:
            tensors.result()
    if verbose:
        for s, log in zip(srcs, logs):
            if log.strip():
                print(f"--- {os.path.basename(s)}\n{log}", file=sys.stderr)
    tmp = LIB + ".tmp"
    cmd = [nvcc, "-gencode", "arch=compute_100a,code=sm_100a", "-shared", "-o", tmp, *objs, "-lcudart"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError("link failed:\n" + r.stderr)
    os.replace(tmp, LIB)
    return LIB


if __name__ == "__main__":
    v = "-v" in sys.argv
    xs = ["-Xptxas", "-v"] if "--ptxas-v" in sys.argv else []
    print(build(force="-f" in sys.argv or bool(xs), verbose=v or bool(xs), extra_flags=xs))
