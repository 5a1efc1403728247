"""Build the in-tree CUDA library ``libmurm_b200.so`` for sm_100a and its torch binding.

    python -m murmurative_attention_b200.build

Compiles every ``csrc/*.cu`` with nvcc for ``sm_100a`` only and links one
shared library next to this file. The library exports the C ABI declared in
``include/murm.h``; the Python package loads it with ctypes. ``csrc/murm_torch.cpp``
(the block operators' argument checks and autograd nodes, over the same C ABI)
is compiled with the host compiler against the installed torch into
``_murm_torch.so`` beside it.
"""
from __future__ import annotations

import glob
import os
import shutil
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
LIB = os.path.join(HERE, "libmurm_b200.so")
BINDING = os.path.join(HERE, "_murm_torch.so")
BINDING_SOURCE = os.path.join(HERE, "csrc", "murm_torch.cpp")
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ["-O3", "-std=c++17", "-lineinfo", "--expt-relaxed-constexpr", "-Xcompiler", "-fPIC",
              "-Xcompiler", "-O3", "-Xcompiler", "-fvisibility=hidden"]


def _nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found: set NVCC or put the CUDA toolkit's bin/ on PATH")


def sources():
    return sorted(glob.glob(os.path.join(HERE, "csrc", "*.cu")))


def headers():
    return sorted(glob.glob(os.path.join(HERE, "csrc", "*.cuh")) +
                  glob.glob(os.path.join(ROOT, "include", "*.h")))


def up_to_date() -> bool:
    if not os.path.exists(LIB):
        return False
    t = os.path.getmtime(LIB)
    return all(os.path.getmtime(p) <= t for p in sources() + headers())


def build_binding(force: bool = False, verbose: bool = False) -> str:
    """The torch binding: plain C++ on the C ABI's header, no CUDA code of its own."""
    header = os.path.join(ROOT, "include", "murm.h")
    if not force and os.path.exists(BINDING) and \
            os.path.getmtime(BINDING) >= max(os.path.getmtime(p) for p in (BINDING_SOURCE, header)):
        return BINDING
    import torch
    base = os.path.dirname(torch.__file__)
    cuda = os.path.dirname(os.path.dirname(os.path.realpath(_nvcc())))
    includes = [os.path.join(base, "include"), os.path.join(base, "include", "torch", "csrc", "api", "include"),
                os.path.join(cuda, "include"), sysconfig.get_paths()["include"]]
    tmp = BINDING + ".tmp"
    # nvcc's own host compiler: torch shares its C++ runtime, a compiler that links another one
    # statically gives a library whose streams and exceptions do not mix with torch's
    cmd = [shutil.which("g++") or "g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", "-DTORCH_EXTENSION_NAME=_murm_torch",
           "-I", os.path.join(ROOT, "include")]
    for path in includes:
        cmd += ["-isystem", path]
    cmd += [BINDING_SOURCE, "-o", tmp, "-L", os.path.join(base, "lib"), "-ltorch", "-ltorch_cpu", "-ltorch_python",
            "-lc10", "-lc10_cuda"]
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.run(cmd, check=True)
    os.replace(tmp, BINDING)
    return BINDING


def build(force: bool = False, verbose: bool = False, extra_flags=()) -> str:
    build_binding(force, verbose)
    if not force and up_to_date():
        return LIB
    nvcc = _nvcc()
    objdir = os.path.join(HERE, "_build")
    os.makedirs(objdir, exist_ok=True)
    objs = []
    for src in sources():
        obj = os.path.join(objdir, os.path.basename(src)[:-3] + ".o")
        cmd = [nvcc, *ARCH, *NVCC_FLAGS, *extra_flags, "-I", os.path.join(ROOT, "include"), "-dc", src, "-o", obj]
        if verbose:
            print(" ".join(cmd), flush=True)
        subprocess.run(cmd, check=True)
        objs.append(obj)
    tmp = LIB + ".tmp"
    cmd = [nvcc, *ARCH, "-shared", "-Xcompiler", "-fPIC", *objs, "-o", tmp, "-lcudart"]
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.run(cmd, check=True)
    os.replace(tmp, LIB)
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose=True))
