"""Build the sm_100a CUDA library ``libscalesweep_b200.so`` in-tree, and beside it
``_kv_binding.so``, the Python binding of the KV-cache operators (host code
against torch's headers, linked to the library).

    python -m test_speed_scalesweep_b200.build [--force]

nvcc cross-compiles for ``-gencode arch=compute_100a,code=sm_100a`` without a
GPU.  The library links the CUDA runtime dynamically (``-cudart shared``), so
inside a PyTorch process it shares torch's already-loaded libcudart.
"""
from __future__ import annotations

import glob
import os
import shutil
import subprocess
import sys

PKG = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG)
CSRC = os.path.join(PKG, "csrc")
INCLUDE = os.path.join(ROOT, "include")
LIB_NAME = "libscalesweep_b200.so"
LIB_PATH = os.path.join(PKG, LIB_NAME)
BUILD_DIR = os.path.join(PKG, "_build")
BINDING_SRC = os.path.join(CSRC, "kv_binding.cpp")
BINDING_PATH = os.path.join(PKG, "_kv_binding.so")

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ["-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC", "-Xcompiler", "-Wall",
              "--expt-relaxed-constexpr", "-Xptxas", "-warn-spills"]


def _nvcc() -> str:
    cand = os.environ.get("NVCC") or shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    return cand


def sources() -> list[str]:
    return sorted(glob.glob(os.path.join(CSRC, "*.cu")))


def _deps() -> list[str]:
    return (sources() + glob.glob(os.path.join(CSRC, "*.cuh")) +
            glob.glob(os.path.join(INCLUDE, "*.h")))


def up_to_date() -> bool:
    if not os.path.exists(LIB_PATH):
        return False
    t = os.path.getmtime(LIB_PATH)
    if not all(os.path.getmtime(d) <= t for d in _deps()):
        return False
    return (os.path.exists(BINDING_PATH)
            and os.path.getmtime(BINDING_PATH) >= max(t, os.path.getmtime(BINDING_SRC)))


def build_binding(verbose: bool = False) -> None:
    import sysconfig

    import torch
    root = os.path.dirname(torch.__file__)
    cuda = os.path.dirname(os.path.dirname(os.path.realpath(_nvcc())))
    tmp = BINDING_PATH + ".tmp"
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared", "-Wall",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}",
           "-isystem", sysconfig.get_paths()["include"],
           "-isystem", os.path.join(root, "include"),
           "-isystem", os.path.join(root, "include", "torch", "csrc", "api", "include"),
           "-isystem", os.path.join(cuda, "include"), BINDING_SRC, "-o", tmp,
           "-L", PKG, f"-l:{LIB_NAME}", "-L", os.path.join(root, "lib"), "-ltorch_python",
           "-ltorch_cpu", "-ltorch_cuda", "-lc10", "-lc10_cuda", "-Wl,-rpath,$ORIGIN"]
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.check_call(cmd)
    os.replace(tmp, BINDING_PATH)


def build(force: bool = False, verbose: bool = False) -> str:
    if not force and up_to_date():
        return LIB_PATH
    os.makedirs(BUILD_DIR, exist_ok=True)
    nvcc = _nvcc()
    if all(os.path.exists(f) for f in (LIB_PATH, BINDING_PATH)) and not force:
        # only the binding's source is newer
        lib_time = os.path.getmtime(LIB_PATH)
        if all(os.path.getmtime(d) <= lib_time for d in _deps()):
            build_binding(verbose)
            return LIB_PATH
    objs = []
    for src in sources():
        obj = os.path.join(BUILD_DIR, os.path.basename(src)[:-3] + ".o")
        cmd = [nvcc, *ARCH, *NVCC_FLAGS, "-I", INCLUDE, "-c", src, "-o", obj]
        if verbose:
            cmd += ["-Xptxas", "-v"]
            print(" ".join(cmd), flush=True)
        subprocess.check_call(cmd)
        objs.append(obj)
    tmp = LIB_PATH + ".tmp"
    cuda_lib = os.path.join(os.path.dirname(os.path.dirname(os.path.realpath(nvcc))), "lib64")
    cmd = [nvcc, *ARCH, "-shared", "-cudart", "shared", "-o", tmp, *objs,
           "-Xlinker", "-rpath=" + cuda_lib]
    subprocess.check_call(cmd)
    os.replace(tmp, LIB_PATH)
    build_binding(verbose)
    return LIB_PATH


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
