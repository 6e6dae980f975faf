"""Build libzs.so (all sm_100a kernels + the C ABI) in-tree with nvcc.

The library is a plain shared object: no torch headers, no Python API.  It is
written next to this file so it travels with the source tree.  Beside it
_paged.so, a small host-only binding of the paged cache operators to CPython and
torch, is compiled with g++ and linked against it; _paged.so.abi names the Python and
torch that it fits (it says so itself, too, when it is loaded).
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sysconfig
from pathlib import Path

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent
CSRC = ROOT / "csrc"
INCLUDE = ROOT.parent / "include"
LIB = PKG / "libzs.so"
BINDING = PKG / "_paged.so"
BINDING_ABI = PKG / "_paged.so.abi"     # what BINDING was compiled against

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-lineinfo", "-std=c++17",
    "-shared", "-Xcompiler", "-fPIC",
    "--expt-relaxed-constexpr",
]


def _nvcc() -> str:
    cand = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not Path(cand).exists():
        raise RuntimeError("nvcc not found: the zs CUDA library cannot be built")
    return cand


def sources():
    return sorted(CSRC.glob("*.cu")) + sorted(CSRC.glob("*.cuh")) + [INCLUDE / "zs.h"]


def needs_build() -> bool:
    if not LIB.exists():
        return True
    t = LIB.stat().st_mtime
    return any(p.stat().st_mtime > t for p in sources())


def binding_abi() -> str:
    """The interpreter and torch whose C++ interfaces the binding is compiled against."""
    import torch

    return (f"{sysconfig.get_config_var('SOABI')} torch {torch.__version__} "
            f"cxx11abi {int(torch._C._GLIBCXX_USE_CXX11_ABI)}")


def binding_needs_build() -> bool:
    if not BINDING.exists() or not BINDING_ABI.exists() or BINDING_ABI.read_text() != binding_abi():
        return True
    t = BINDING.stat().st_mtime
    return any(p.stat().st_mtime > t for p in (CSRC / "zs_paged_py.cpp", INCLUDE / "zs.h"))


def build_binding(force: bool = False, verbose: bool = False) -> Path:
    if not force and not binding_needs_build():
        return BINDING
    import torch

    cxx = shutil.which("g++")
    if cxx is None:
        raise RuntimeError("g++ not found: the paged operators' binding cannot be built")
    t = Path(torch.__file__).resolve().parent
    cuda = Path(_nvcc()).resolve().parent.parent
    tmp = BINDING.with_suffix(".so.tmp")
    cmd = [cxx, "-O2", "-std=c++17", "-shared", "-fPIC", f'-DZS_BINDING_ABI="{binding_abi()}"',
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", "-I", str(INCLUDE),
           "-I", sysconfig.get_paths()["include"], "-I", str(t / "include"),
           "-I", str(t / "include" / "torch" / "csrc" / "api" / "include"), "-I", str(cuda / "include"),
           "-o", str(tmp), str(CSRC / "zs_paged_py.cpp"), "-L", str(PKG), "-l:libzs.so", "-L", str(t / "lib"),
           "-lc10", "-lc10_cuda", "-ltorch", "-ltorch_cpu", "-ltorch_python", "-Wl,-rpath,$ORIGIN"]
    if verbose:
        print(" ".join(cmd))
    subprocess.run(cmd, check=True)
    BINDING_ABI.unlink(missing_ok=True)   # no moment at which it speaks of another binary
    os.replace(tmp, BINDING)
    BINDING_ABI.write_text(binding_abi())
    return BINDING


def build(force: bool = False, verbose: bool = False) -> Path:
    if force or needs_build():
        tmp = LIB.with_suffix(".so.tmp")
        cmd = [_nvcc(), *NVCC_FLAGS, "-I", str(INCLUDE), "-o", str(tmp), str(CSRC / "zs_lib.cu")]
        if verbose:
            print(" ".join(cmd))
        subprocess.run(cmd, check=True)
        os.replace(tmp, LIB)
    build_binding(force, verbose)
    return LIB


if __name__ == "__main__":
    build(force=True, verbose=True)
    print(LIB)
