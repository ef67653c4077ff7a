"""Builds libkea_lowbit.so (sm_100a) into the kea_kernels package directory with nvcc.

Usage: python kea-kernels_b200/build.py [--force]
The library is compiled in-tree so it travels with the source tree; nothing is JIT-compiled at run time.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
import tempfile
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

HERE = Path(__file__).resolve().parent
ROOT = HERE.parent
CSRC = HERE / "csrc"
OUT = HERE / "kea_kernels" / "libkea_lowbit.so"
SOURCES = [CSRC / f"{name}.cu" for name in ("kea_lowbit", "int8_gemm", "residual_norm", "beam")]
HEADERS = sorted(CSRC.glob("*.cuh")) + [CSRC / "host.h", ROOT / "include" / "kea_lowbit.h"]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("nvcc not found: set NVCC or add the CUDA toolkit to PATH")


def compile_command(source: Path, obj: Path) -> list[str]:
    return [nvcc(), "-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17",
            "-fmad=false", "-Xptxas", "-v", f"-I{ROOT / 'include'}", "-Xcompiler", "-fPIC,-O2", "-c",
            "-o", str(obj), str(source)]


def link_command(objects: list[Path]) -> list[str]:
    return [nvcc(), "-gencode", "arch=compute_100a,code=sm_100a", "-shared", "-o", str(OUT), *map(str, objects)]


def newest_input(source: Path) -> float:
    return max(p.stat().st_mtime for p in [source, *HEADERS, Path(__file__)])


def stale() -> bool:
    return not OUT.exists() or any(newest_input(s) > OUT.stat().st_mtime for s in SOURCES)


def run(cmd: list[str]) -> str:
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"nvcc failed ({res.returncode}):\n{res.stdout}\n{res.stderr}")
    return res.stderr


def build(force: bool = False, verbose: bool = False) -> Path:
    """Compiles the sources side by side into a temporary folder and links them."""
    if force or stale():
        with tempfile.TemporaryDirectory() as tmp, ThreadPoolExecutor(len(SOURCES)) as pool:
            objects = [Path(tmp) / f"{s.stem}.o" for s in SOURCES]
            logs = list(pool.map(run, map(compile_command, SOURCES, objects)))
            logs.append(run(link_command(objects)))
        if verbose:
            print("".join(logs))
    return OUT


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose=True))
