"""Build libdcr_b200.so (the sm_100a CUDA library behind the C ABI in include/dcr_b200.h) and
dcr_b200_torch.so (the paged operators' binding to torch tensors, csrc/dcr_torch.cpp).

The library is one nvcc translation unit (csrc/dcr_b200_lib.cu) built in-tree into
``dcr_b200/lib/libdcr_b200.so`` with ``-gencode arch=compute_100a,code=sm_100a``.
It links the CUDA runtime statically and reaches the driver's tensor-map encoder through
``cudaGetDriverEntryPoint``, so it needs neither ``-lcuda`` nor a matching libcudart at
run time.

Usage: ``python -m dcr_b200.build [--force] [--no-binding]`` (with ``dcr-attention_v3_b200`` on
sys.path). The binding is built where torch is installed; ``--no-binding`` leaves it out.
"""
from __future__ import annotations

import glob
import importlib.util
import os
import shutil
import subprocess
import sys

PKG_DIR = os.path.dirname(os.path.abspath(__file__))
SRC_ROOT = os.path.dirname(PKG_DIR)                 # dcr-attention_v3_b200/
REPO_ROOT = os.path.dirname(SRC_ROOT)
CSRC = os.path.join(SRC_ROOT, "csrc")
INCLUDE = os.path.join(REPO_ROOT, "include")
LIB_DIR = os.path.join(PKG_DIR, "lib")
LIB_PATH = os.path.join(LIB_DIR, "libdcr_b200.so")
TORCH_PATH = os.path.join(LIB_DIR, "dcr_b200_torch.so")
TORCH_SOURCE = os.path.join(CSRC, "dcr_torch.cpp")
TORCH_STAMP = os.path.join(LIB_DIR, "dcr_b200_torch.stamp")  # what the binding was built for

ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ["-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC", "-shared",
              "--expt-relaxed-constexpr", "-Xptxas", "-warn-spills"]


def nvcc_path() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found: the CUDA 12.9 toolkit is required to build libdcr_b200")


def _sources():
    return sorted(glob.glob(os.path.join(CSRC, "*.cu")) + glob.glob(os.path.join(CSRC, "*.cuh"))
                  + glob.glob(os.path.join(CSRC, "*.h")) + [os.path.join(INCLUDE, "dcr_b200.h")])


def up_to_date() -> bool:
    if not os.path.exists(LIB_PATH):
        return False
    t = os.path.getmtime(LIB_PATH)
    return all(os.path.getmtime(s) <= t for s in _sources())


def build_torch(force: bool = False, verbose: bool = False) -> str:
    """Compile the torch binding (host code only) if a source is newer than it, or if it was built
    for another torch or Python."""
    import torch
    stamp = f"{torch.__version__} {sys.implementation.cache_tag}"
    sources = [TORCH_SOURCE, os.path.join(CSRC, "dcr_tables.h"), os.path.join(INCLUDE, "dcr_b200.h")]
    if not force and os.path.exists(TORCH_PATH) and _stamp() == stamp and all(
            os.path.getmtime(s) <= os.path.getmtime(TORCH_PATH) for s in sources):
        return TORCH_PATH
    import sysconfig

    from torch.utils.cpp_extension import include_paths, library_paths
    cuda_include = os.path.join(os.path.dirname(os.path.dirname(nvcc_path())), "include")
    includes = [INCLUDE, *include_paths(), cuda_include, sysconfig.get_path("include")]
    tmp = TORCH_PATH + ".tmp"
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared",
           "-fvisibility=hidden",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           *(f"-isystem{i}" for i in includes), TORCH_SOURCE, "-o", tmp, f"-L{LIB_DIR}",
           "-l:libdcr_b200.so", *(f"-L{d}" for d in library_paths()), "-lc10", "-lc10_cuda",
           "-ltorch_cpu", "-ltorch_python", "-Wl,-rpath,$ORIGIN"]
    if verbose:
        print(" ".join(cmd), file=sys.stderr)
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"the torch binding failed to build ({r.returncode}):\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, TORCH_PATH)
    with open(TORCH_STAMP, "w") as f:
        f.write(stamp)
    return TORCH_PATH


def _stamp() -> str:
    try:
        with open(TORCH_STAMP) as f:
            return f.read()
    except OSError:
        return ""


def build(force: bool = False, verbose: bool = False, binding: bool = True) -> str:
    """Compile the libraries if any of their sources is newer; return libdcr_b200.so's path. The
    torch binding is left out without ``binding`` or where torch is not installed."""
    if force or not up_to_date():
        _build_library(verbose)
    if binding and importlib.util.find_spec("torch") is not None:
        build_torch(force, verbose)
    return LIB_PATH


def _build_library(verbose: bool) -> None:
    os.makedirs(LIB_DIR, exist_ok=True)
    tmp = LIB_PATH + ".tmp"
    cmd = [nvcc_path(), *ARCH_FLAGS, *NVCC_FLAGS, f"-I{INCLUDE}", f"-I{CSRC}",
           os.path.join(CSRC, "dcr_b200_lib.cu"), "-o", tmp]
    if verbose:
        print(" ".join(cmd), file=sys.stderr)
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"nvcc failed ({r.returncode}):\n{r.stdout}\n{r.stderr}")
    if "spill" in (r.stderr or "") and verbose:
        print(r.stderr, file=sys.stderr)
    os.replace(tmp, LIB_PATH)


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose=True, binding="--no-binding" not in sys.argv))
