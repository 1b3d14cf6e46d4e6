"""Builds torchisotonic_b200/libtiso.so: the CUDA kernels behind include/tiso.h, for sm_100a; and
torchisotonic_b200/_native.so, the extension module over it that the losses and the optimizer step
are called through.

    python -m torchisotonic_b200.build [--verbose]

nvcc compiles for the B200 (compute_100a / sm_100a) only; no JIT build at import time.
"""

from __future__ import annotations

import os
import shutil
import subprocess
import sys
import sysconfig
from pathlib import Path

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent
CSRC = PKG / "csrc"
LIB = PKG / "libtiso.so"
SOURCES = [CSRC / f for f in ("tiso.cu", "calib.cu", "logits.cu", "preference.cu", "adamw.cu")]
NATIVE, NATIVE_SOURCE = PKG / "_native.so", CSRC / "native.cpp"
DEPS = SOURCES + sorted(CSRC.glob("*.cuh")) + [ROOT / "include" / "tiso.h"]

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-lineinfo", "-std=c++17",
    "-Xcompiler", "-fPIC", "-shared",
    "--expt-relaxed-constexpr",
    "-Xptxas", "-warn-spills",
]


def nvcc() -> str:
    cuda = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    path = Path(cuda) / "bin" / "nvcc"
    return str(path) if path.exists() else (shutil.which("nvcc") or "nvcc")


def stale(built: Path = LIB, deps: list[Path] = DEPS) -> bool:
    return not built.exists() or any(p.stat().st_mtime > built.stat().st_mtime for p in deps)


def build(force: bool = False, verbose: bool = False) -> Path:
    if force or stale():
        tmp = LIB.with_suffix(".so.tmp")
        cmd = [nvcc(), *NVCC_FLAGS, *(["-Xptxas", "-v"] if verbose else []),
               "-o", str(tmp), *map(str, SOURCES), "-lcudart"]
        subprocess.run(cmd, check=True, cwd=str(ROOT))
        tmp.replace(LIB)
    build_native(force)
    return LIB


def build_native(force: bool = False) -> Path:
    """The extension module, against this interpreter's torch; it finds libtiso.so beside itself."""
    if not force and not stale(NATIVE, [NATIVE_SOURCE, ROOT / "include" / "tiso.h"]):
        return NATIVE
    from torch.utils import cpp_extension

    cuda = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    includes = [*cpp_extension.include_paths(), f"{cuda}/include", sysconfig.get_path("include")]
    tmp = NATIVE.with_suffix(".so.tmp")
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared",
           *(f"-I{p}" for p in includes), str(NATIVE_SOURCE), "-o", str(tmp),
           *(f"-L{p}" for p in cpp_extension.library_paths()), f"-L{PKG}",
           "-ltorch", "-ltorch_cpu", "-ltorch_python", "-lc10", "-lc10_cuda", "-l:libtiso.so",
           "-Wl,-rpath,$ORIGIN"]
    subprocess.run(cmd, check=True, cwd=str(ROOT))
    tmp.replace(NATIVE)
    return NATIVE


if __name__ == "__main__":
    build(force=True, verbose="--verbose" in sys.argv)
    print(LIB)
