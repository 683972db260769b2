"""Build libixb200.so in-tree for sm_100a (nvcc; no GPU needed to compile), and beside it the torch
binding of the fp8 linears, ``_ixb_torch.so`` (host C++ against the installed torch's headers).

``python -m ignite_xdna_b200.build`` or ``ignite_xdna_b200.build.build()``.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
from pathlib import Path

PKG = Path(__file__).resolve().parent
CSRC = PKG / "csrc"
OUT = PKG / "libixb200.so"
BINDING = PKG / "_ixb_torch.so"
BINDING_SRC = CSRC / "ixb_torch.cpp"
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC", "-shared", "--expt-relaxed-constexpr"]


def nvcc() -> str:
    cand = [os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"]
    for c in cand:
        if c and Path(c).exists():
            return c
    raise RuntimeError("nvcc not found")


def sources():
    return sorted(CSRC.glob("*.cu")) + sorted(CSRC.glob("*.cuh")) + [PKG.parent / "include" / "ixb200.h"]


def up_to_date() -> bool:
    if not OUT.exists():
        return False
    t = OUT.stat().st_mtime
    return all(s.stat().st_mtime <= t for s in sources())


def build(force: bool = False, verbose: bool = False) -> Path:
    if not force and up_to_date():
        return OUT
    tmp = OUT.with_suffix(f".tmp{os.getpid()}.so")
    cmd = [nvcc(), *ARCH, *FLAGS, "-o", str(tmp), str(CSRC / "ixb_api.cu")]
    if verbose:
        cmd.insert(1, "-Xptxas=-v")
    r = subprocess.run(cmd, cwd=CSRC, capture_output=True, text=True)
    if r.returncode != 0:
        sys.stderr.write(r.stdout + r.stderr)
        raise RuntimeError("nvcc failed building libixb200.so")
    if verbose:
        sys.stderr.write(r.stderr)
    os.replace(tmp, OUT)
    return OUT


def build_binding(force: bool = False) -> Path:
    import sysconfig

    import torch
    src = [BINDING_SRC, PKG.parent / "include" / "ixb200.h", Path(torch.__file__)]
    if not force and BINDING.exists() and all(s.stat().st_mtime <= BINDING.stat().st_mtime for s in src):
        return BINDING
    root = Path(torch.__file__).resolve().parent
    cuda = Path(nvcc()).resolve().parent.parent
    tmp = BINDING.with_suffix(f".tmp{os.getpid()}.so")
    inc = [root / "include", root / "include" / "torch" / "csrc" / "api" / "include", cuda / "include",
           sysconfig.get_paths()["include"]]
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}", *[f"-I{p}" for p in inc], str(BINDING_SRC),
           "-o", str(tmp), f"-L{root / 'lib'}", "-ltorch_python", "-ltorch_cuda", "-ltorch_cpu", "-lc10", "-lc10_cuda"]
    r = subprocess.run(cmd, cwd=CSRC, capture_output=True, text=True)
    if r.returncode != 0:
        sys.stderr.write(r.stdout + r.stderr)
        raise RuntimeError("building the torch binding failed")
    os.replace(tmp, BINDING)
    return BINDING


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
    print(build_binding(force="--force" in sys.argv))
