"""Builds ``libmole_b200.so`` in-tree with nvcc for sm_100a.

Run as ``python mole_b200/build.py`` (add ``-v`` for ptxas resource usage); it is loaded by path,
not through the package, because importing the package needs the library it builds.  The library is
a plain C-ABI shared object: no torch headers, no pybind.  Beside it goes a small extension module with
the host side of the calls whose checks would take longer in Python than they do on the GPU.
"""
from __future__ import annotations

import importlib.metadata
import importlib.util
import os
import shutil
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

HERE = Path(__file__).resolve().parent
CSRC = HERE / "csrc"
OUT_DIR = HERE / "lib"
LIB = OUT_DIR / "libmole_b200.so"
HOST_LIB = OUT_DIR / "_host.so"          # extension module over torch's tensors (host.cpp)
HOST_STAMP = OUT_DIR / "_host.built_for"  # the Python and torch that it was built for
SOURCES = ["route.cu", "dispatch.cu", "gate_mma.cu", "gemm_simt.cu", "gemm_tc.cu", "ffn.cu", "runtime.cu", "adam.cu",
           "adam_multi.cu", "ragged.cu", "ragged_simt.cu", "ragged_tc.cu", "ragged_few.cu"]
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]


def _nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("nvcc not found; the CUDA library cannot be built")


def _nccl_include() -> list[str]:
    site = Path(sysconfig.get_paths()["purelib"]) / "nvidia" / "nccl" / "include"
    return ["-I", str(site)] if (site / "nccl.h").exists() else []


def host_abi() -> str:
    """What the extension module has to be built for: this Python and this torch."""
    try:
        torch = importlib.metadata.version("torch")
    except importlib.metadata.PackageNotFoundError:      # a source tree
        torch = "of a source tree"
    return f"{sys.implementation.cache_tag}, torch {torch}"


def _build_host(nvcc: str) -> None:
    # by way of nvcc, so that the compiler is the one the library is built with: $CXX may be a tool chain
    # whose modules crash under torch
    torch = Path(importlib.util.find_spec("torch").submodule_search_locations[0])
    cmd = [nvcc, "-x", "c++", "-O2", "-std=c++20", "-shared", "-Xcompiler", "-fPIC,-fvisibility=hidden",
           "-I", str(torch / "include"), "-I", str(torch / "include/torch/csrc/api/include"),
           "-I", sysconfig.get_paths()["include"], str(CSRC / "host.cpp"), "-o", str(HOST_LIB),
           "-L", str(torch / "lib"), "-ltorch_python", "-ltorch_cpu", "-lc10", "-lc10_cuda"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        sys.stderr.write(res.stdout + res.stderr)
        raise RuntimeError("building _host.so failed")
    HOST_STAMP.write_text(host_abi())


def _stale() -> bool:
    if not LIB.exists() or not HOST_LIB.exists():
        return True
    if not HOST_STAMP.exists() or HOST_STAMP.read_text() != host_abi():
        return True
    newest = max(p.stat().st_mtime for p in list(CSRC.iterdir()) + [HERE.parent / "include" / "mole_b200.h"])
    return newest > min(LIB.stat().st_mtime, HOST_LIB.stat().st_mtime)


def build(verbose: bool = False, force: bool = False) -> Path:
    if not force and not _stale():
        return LIB
    nvcc = _nvcc()
    OUT_DIR.mkdir(exist_ok=True)
    obj_dir = HERE / "_obj"
    obj_dir.mkdir(exist_ok=True)
    common = [nvcc, *ARCH, "-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC",
              "--expt-relaxed-constexpr", *_nccl_include()]
    if verbose:
        common += ["-Xptxas", "-v"]

    def compile_one(src: str) -> Path:
        obj = obj_dir / (src + ".o")
        cmd = common + ["-c", str(CSRC / src), "-o", str(obj)]
        res = subprocess.run(cmd, capture_output=True, text=True)
        if verbose or res.returncode != 0:
            sys.stderr.write(f"--- {src}\n{res.stdout}{res.stderr}")
        if res.returncode != 0:
            raise RuntimeError(f"nvcc failed on {src}")
        return obj

    with ThreadPoolExecutor(max_workers=min(len(SOURCES) + 1, os.cpu_count() or 1)) as pool:
        host = pool.submit(_build_host, nvcc)
        objs = list(pool.map(compile_one, SOURCES))
        host.result()
    link = [nvcc, *ARCH, "-shared", "-o", str(LIB), *map(str, objs), "-ldl"]
    res = subprocess.run(link, capture_output=True, text=True)
    if res.returncode != 0:
        sys.stderr.write(res.stdout + res.stderr)
        raise RuntimeError("linking libmole_b200.so failed")
    return LIB


if __name__ == "__main__":
    path = build(verbose="-v" in sys.argv, force=True)
    print(path)
