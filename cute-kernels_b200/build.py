"""Builds libfma_b200.so (the C-ABI library of sm_100a kernels) in-tree with nvcc, and fma_b200_torch.so (the torch
binding of the 8-bit operators, which calls it) with g++.

Usage:  python cute-kernels_b200/build.py [--force] [--verbose]

The library is compiled for sm_100a only (explicit -gencode; the -arch=sm_100a shorthand also
emits generic compute_100 PTX, which rejects tcgen05).  Objects and the .so stay next to the
sources; nothing is installed outside the tree.
"""

from __future__ import annotations

import argparse
import os
import shutil
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

ROOT = Path(__file__).resolve().parent
CSRC = ROOT / "csrc"
OUT_DIR = ROOT / "fma_b200" / "_lib"
LIB_PATH = OUT_DIR / "libfma_b200.so"
BINDING_PATH = OUT_DIR / "fma_b200_torch.so"
HEADER = ROOT.parent / "include" / "fma_b200.h"

NVCC_FLAGS = [
    "-gencode",
    "arch=compute_100a,code=sm_100a",
    "-O3",
    "-std=c++17",
    "-lineinfo",
    "-Xcompiler",
    "-fPIC",
    "--expt-relaxed-constexpr",
]


def _nvcc() -> str:
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(nvcc):
        raise RuntimeError("nvcc not found; the CUDA kernels cannot be built")
    return nvcc


def _cxx() -> str:
    """The system's compiler, whatever CXX says: one with a newer C++ library of its own links parts of that library into
    the binding, next to the one that torch has loaded."""
    for cxx in ("/usr/bin/g++", shutil.which("g++")):
        if cxx and os.path.exists(cxx):
            return cxx
    raise RuntimeError("g++ not found; the torch binding cannot be built")


def _stale(target: Path, deps: list[Path]) -> bool:
    if not target.exists():
        return True
    t = target.stat().st_mtime
    return any(d.stat().st_mtime > t for d in deps)


def build_binding(force: bool = False) -> Path:
    """Compiles csrc/torch_fp8.cpp against the installed torch; libfma_b200.so has to be there."""
    source = CSRC / "torch_fp8.cpp"
    if not (force or _stale(BINDING_PATH, [source, HEADER, Path(__file__)])):
        return BINDING_PATH
    import torch

    base = Path(torch.__file__).resolve().parent
    cuda = Path(_nvcc()).resolve().parent.parent
    include = [base / "include", base / "include" / "torch" / "csrc" / "api" / "include", cuda / "include", sysconfig.get_paths()["include"]]
    cmd = [
        _cxx(), "-O2", "-std=c++17", "-fPIC", "-shared", *[f"-I{p}" for p in include],
        f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", f"-DTORCH_EXTENSION_NAME={BINDING_PATH.stem}",
        str(source), "-o", str(BINDING_PATH), f"-L{base / 'lib'}", "-lc10", "-ltorch_cpu", "-ltorch", "-ltorch_python", "-lc10_cuda",
        "-ltorch_cuda", f"-L{OUT_DIR}", f"-l:{LIB_PATH.name}", "-Wl,-rpath,$ORIGIN",
    ]  # fmt: skip
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        sys.stderr.write(res.stdout + res.stderr)
        raise RuntimeError("building the torch binding failed")
    return BINDING_PATH


def build_library(force: bool = False, verbose: bool = False) -> Path:
    """Compiles every csrc/*.cu, links libfma_b200.so and builds the torch binding; returns the library's path."""
    nvcc = _nvcc()
    OUT_DIR.mkdir(parents=True, exist_ok=True)
    sources = sorted(CSRC.glob("*.cu"))
    headers = sorted(CSRC.glob("*.cuh")) + [HEADER, Path(__file__)]
    obj_dir = OUT_DIR / "obj"
    obj_dir.mkdir(exist_ok=True)

    def compile_one(src: Path) -> Path:
        obj = obj_dir / (src.stem + ".o")
        if force or _stale(obj, [src] + headers):
            cmd = [nvcc, *NVCC_FLAGS, "-c", str(src), "-o", str(obj)]
            if verbose:
                cmd.insert(1, "-Xptxas")
                cmd.insert(2, "-v")
            res = subprocess.run(cmd, capture_output=True, text=True)
            if verbose or res.returncode != 0:
                sys.stderr.write(res.stdout + res.stderr)
            if res.returncode != 0:
                raise RuntimeError(f"nvcc failed on {src.name}")
        return obj

    with ThreadPoolExecutor(max_workers=min(8, len(sources))) as pool:
        objects = list(pool.map(compile_one, sources))

    if force or _stale(LIB_PATH, objects):
        # Export only the fma_b200_* entry points (the driver entry point for tensor maps is
        # resolved at run time through cudaGetDriverEntryPoint, so libcuda is not linked).
        vers = OUT_DIR / "exports.map"
        vers.write_text("{ global: fma_b200_*; local: *; };\n")
        cmd = [
            nvcc,
            "-shared",
            "-gencode",
            "arch=compute_100a,code=sm_100a",
            "-o",
            str(LIB_PATH),
            *[str(o) for o in objects],
            "-Xlinker",
            f"--version-script={vers}",
        ]
        res = subprocess.run(cmd, capture_output=True, text=True)
        if res.returncode != 0:
            sys.stderr.write(res.stdout + res.stderr)
            raise RuntimeError("linking libfma_b200.so failed")
    build_binding(force)
    return LIB_PATH


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--verbose", action="store_true")
    args = ap.parse_args()
    print(build_library(force=args.force, verbose=args.verbose))
