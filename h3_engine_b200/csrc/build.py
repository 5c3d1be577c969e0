"""Build libh3b.so (sm_100a) in-tree with nvcc, and _h3b_torch.so with g++.

    python -m h3_engine_b200.csrc.build [--verbose]

The library is one translation unit (h3b.cu includes every kernel header) so
all kernels share the device error word.  cudart is linked statically: the
library only needs the CUDA driver at run time.  _h3b_torch.so holds the torch
operators that are written in C++; it links libh3b.so and torch.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
from pathlib import Path

HERE = Path(__file__).resolve().parent
PKG = HERE.parent
ROOT = PKG.parent
LIB = PKG / "libh3b.so"
EXT = PKG / "_h3b_torch.so"

ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = [
    "-O3", "-std=c++17", "-lineinfo", "--expt-relaxed-constexpr",
    "-Xcompiler", "-fPIC,-O3,-fvisibility=hidden",
    "-cudart", "static",
]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", shutil.which("nvcc")):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("nvcc not found")


def cxx() -> str:
    """The system's g++, whose C++ runtime is the one that torch loads at run
    time (a newer compiler named by $CXX links parts of its own runtime in,
    and the two crash on each other's streams)."""
    for cand in ("/usr/bin/g++", shutil.which("g++")):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("g++ not found")


def sources() -> list[Path]:
    return sorted(list(HERE.glob("*.cu")) + list(HERE.glob("*.cuh")) + [ROOT / "include" / "h3b.h"])


def up_to_date() -> bool:
    if not LIB.exists():
        return False
    t = LIB.stat().st_mtime
    return all(p.stat().st_mtime <= t for p in sources())


def build(force: bool = False, verbose: bool = False, ptxas_v: bool = False) -> Path:
    if not force and up_to_date():
        return LIB
    tmp = LIB.with_suffix(".so.tmp")
    cmd = [nvcc(), *ARCH_FLAGS, *NVCC_FLAGS, "-shared", "-o", str(tmp), str(HERE / "h3b.cu"),
           "-I", str(ROOT / "include")]
    if ptxas_v:
        cmd += ["-Xptxas", "-v"]
    if verbose:
        print(" ".join(cmd), flush=True)
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        sys.stderr.write(r.stdout + r.stderr)
        raise RuntimeError(f"nvcc failed with exit code {r.returncode}")
    if verbose or ptxas_v:
        sys.stderr.write(r.stderr)
    os.replace(tmp, LIB)
    return LIB


def build_ext(force: bool = False, verbose: bool = False) -> Path:
    """_h3b_torch.so from torch_ext.cpp, against the installed torch and LIB.  A
    file beside it says which torch that was: another one needs another build."""
    import torch
    src = [HERE / "torch_ext.cpp", ROOT / "include" / "h3b.h"]
    abi = int(torch._C._GLIBCXX_USE_CXX11_ABI)
    built_for = f"torch {torch.__version__}, C++11 ABI {abi}\n"
    stamp = EXT.with_suffix(".so.torch")
    if (not force and EXT.exists() and stamp.exists() and stamp.read_text() == built_for
            and all(p.stat().st_mtime <= EXT.stat().st_mtime for p in src)):
        return EXT
    troot = Path(torch.__file__).resolve().parent
    cuda = Path(nvcc()).resolve().parent.parent
    tmp = EXT.with_suffix(".so.tmp")
    cmd = [cxx(), "-O2", "-std=c++17", "-fPIC", "-shared",
           "-fvisibility=hidden", f"-D_GLIBCXX_USE_CXX11_ABI={abi}",
           "-I", str(ROOT / "include"), "-isystem", str(troot / "include"),
           "-isystem", str(cuda / "include"), str(src[0]), "-o", str(tmp),
           "-L", str(PKG), "-lh3b", "-L", str(troot / "lib"), "-lc10", "-lc10_cuda", "-ltorch_cpu",
           "-ltorch_cuda", "-ltorch", "-Wl,-rpath,$ORIGIN"]
    if verbose:
        print(" ".join(cmd), flush=True)
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        sys.stderr.write(r.stdout + r.stderr)
        raise RuntimeError(f"{cmd[0]} failed with exit code {r.returncode}")
    os.replace(tmp, EXT)
    stamp.write_text(built_for)
    return EXT


if __name__ == "__main__":
    build(force="--force" in sys.argv, verbose="--verbose" in sys.argv,
          ptxas_v="--ptxas-v" in sys.argv)
    build_ext(force="--force" in sys.argv, verbose="--verbose" in sys.argv)
    print(LIB)
