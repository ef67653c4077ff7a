"""Builds libkea_lowbit.so (sm_100a, nvcc) and the _binding extension module (g++, against the installed torch) into the
kea_kernels package directory.

Usage: python kea-kernels_b200/build.py [--force]
The library is compiled in-tree so it travels with the source tree; nothing is JIT-compiled at run time.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
import sysconfig
import tempfile
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

HERE = Path(__file__).resolve().parent
ROOT = HERE.parent
CSRC = HERE / "csrc"
OUT = HERE / "kea_kernels" / "libkea_lowbit.so"
BINDING_SOURCE, BINDING = CSRC / "binding.cpp", HERE / "kea_kernels" / "_binding.so"
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


def binding_command() -> list[str]:
    import torch
    from torch.utils import cpp_extension

    cuda = Path(nvcc()).resolve().parents[1] / "include"
    includes = [*cpp_extension.include_paths(), sysconfig.get_paths()["include"], str(cuda), str(ROOT / "include")]
    libs = str(Path(torch.__file__).parent / "lib")
    return [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared",
            f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}", *(f"-I{p}" for p in includes),
            "-o", str(BINDING), str(BINDING_SOURCE), f"-L{libs}", f"-Wl,-rpath,{libs}",
            "-ltorch_python", "-ltorch_cpu", "-ltorch", "-lc10_cuda", "-lc10"]


def newest_input(source: Path) -> float:
    return max(p.stat().st_mtime for p in [source, *HEADERS, Path(__file__)])


def stale() -> bool:
    return not OUT.exists() or any(newest_input(s) > OUT.stat().st_mtime for s in SOURCES)


def binding_stale() -> bool:
    inputs = [BINDING_SOURCE, ROOT / "include" / "kea_lowbit.h", Path(__file__)]
    return not BINDING.exists() or any(p.stat().st_mtime > BINDING.stat().st_mtime for p in inputs)


def run(cmd: list[str]) -> str:
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"{Path(cmd[0]).name} failed ({res.returncode}):\n{res.stdout}\n{res.stderr}")
    return res.stderr


def build_library() -> str:
    """Compiles the sources side by side into a temporary folder and links them."""
    with tempfile.TemporaryDirectory() as tmp, ThreadPoolExecutor(len(SOURCES)) as pool:
        objects = [Path(tmp) / f"{s.stem}.o" for s in SOURCES]
        logs = list(pool.map(run, map(compile_command, SOURCES, objects)))
        return "".join([*logs, run(link_command(objects))])


def build_binding() -> str:
    """Compiles the extension. Without torch there is no Python side to serve, and the library stands alone."""
    try:
        command = binding_command()
    except ModuleNotFoundError as e:
        if e.name != "torch":
            raise
        print("torch is not installed: only the C library is built", file=sys.stderr)
        return ""
    return run(command)


def build(force: bool = False, verbose: bool = False) -> Path:
    """The library, which needs nvcc alone, and the binding beside it. A binding that does not build is an error, after the
    library has been put in its place."""
    library, binding = force or stale(), force or binding_stale()
    with ThreadPoolExecutor(1) as pool:
        extension = pool.submit(build_binding) if binding else None
        log = build_library() if library else ""
        if extension is not None:
            try:
                log += extension.result()
            except Exception as e:
                raise RuntimeError(f"{OUT.name} is built, {BINDING.name} (the Python entry points) is not: {e}") from e
    if verbose:
        print(log)
    return OUT


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose=True))
