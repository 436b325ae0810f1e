"""Build libgfield.so in-tree with nvcc for sm_100a.

The library is plain CUDA C++ behind a C ABI (include/gfield.h); it is built
with explicit nvcc flags (no torch extension machinery) so the same .so can be
loaded from Python (ctypes), C, or any FFI.  It must be built without
--use_fast_math: the renderer relies on CUDA's IEEE expf/log1pf/div/sqrt to
match the reference bit for bit.
"""
from __future__ import annotations

import os
import subprocess
import sys
from pathlib import Path

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent
SOURCES = [PKG / "csrc" / "gfield.cu", PKG / "csrc" / "gfblock.cu"]
HEADERS = [ROOT / "include" / "gfield.h", ROOT / "include" / "gfblock.h", PKG / "csrc" / "tc100.cuh"]
LIB = PKG / "libgfield.so"
# debug build: every shape-derived global access bounds-checked (GF_FLAG_BOUNDS);
# load it instead of the release library with GUASS_B200_LIB=<path>
LIB_CHECK = PKG / "libgfield_check.so"

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-lineinfo", "-std=c++17",
    "-Xcompiler", "-fPIC",
    "-Xptxas", "-warn-spills",
]
OBJECTS = PKG / "build"


def nvcc() -> str:
    cuda = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    cand = Path(cuda) / "bin" / "nvcc"
    return str(cand) if cand.exists() else "nvcc"


def _newer(target: Path, inputs) -> bool:
    """True when ``target`` is missing or older than one of ``inputs``."""
    return not target.exists() or any(p.stat().st_mtime > target.stat().st_mtime for p in inputs)


def needs_build(lib: Path = LIB) -> bool:
    return _newer(lib, SOURCES + HEADERS)


def _object(src: Path, check: bool) -> Path:
    return OBJECTS / (src.stem + ("_check.o" if check else ".o"))


def build(force: bool = False, verbose: bool = False, check: bool = False) -> Path:
    """Build the release library (or, with ``check``, the bounds-checked one):
    one object per source, compiled side by side and kept for the next build."""
    lib = LIB_CHECK if check else LIB
    if not force and not needs_build(lib):
        return lib
    OBJECTS.mkdir(exist_ok=True)
    jobs = []
    for src in SOURCES:
        obj = _object(src, check)
        if force or _newer(obj, [src, *HEADERS]):
            tmp = obj.with_suffix(".tmp.o")
            cmd = [nvcc(), *NVCC_FLAGS, *(["-DGF_CHECK"] if check else []),
                   f"-I{ROOT / 'include'}", "-c", str(src), "-o", str(tmp)]
            if verbose:
                print(" ".join(cmd), file=sys.stderr)
            jobs.append((subprocess.Popen(cmd), cmd, tmp, obj))
    for proc, cmd, tmp, obj in jobs:
        if proc.wait() != 0:
            raise subprocess.CalledProcessError(proc.returncode, cmd)
        os.replace(tmp, obj)
    tmp = lib.with_suffix(".so.tmp")
    cmd = [nvcc(), *NVCC_FLAGS, "-shared", *(str(_object(s, check)) for s in SOURCES), "-o", str(tmp), "-lcudart"]
    if verbose:
        print(" ".join(cmd), file=sys.stderr)
    subprocess.run(cmd, check=True)
    os.replace(tmp, lib)
    return lib


def build_all(force: bool = False, verbose: bool = False) -> list[Path]:
    return [build(force, verbose), build(force, verbose, check=True)]


if __name__ == "__main__":
    for lib in build_all(force="--force" in sys.argv, verbose=True):
        print(lib)
