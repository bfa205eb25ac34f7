"""Builds ``libmuon_b200.so`` (the C-ABI CUDA library) and ``_tables.so`` (the Python extension that makes
its multi-tensor calls from lists of tensors) in-tree, with nvcc for sm_100a and the host compiler.

Usage: ``python muon_b200/build.py [--force] [-v]``. Run it as a script: importing the
package needs the library to exist already. nvcc cross-compiles, so no GPU is needed.
"""
from __future__ import annotations

import importlib.metadata
import importlib.util
import os
import shutil
import subprocess
import sys
import sysconfig
import tempfile
from concurrent.futures import ThreadPoolExecutor

PKG_DIR = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(PKG_DIR, "csrc")
LIB_PATH = os.path.join(PKG_DIR, "libmuon_b200.so")
TABLES_PATH = os.path.join(PKG_DIR, "_tables.so")
TABLES_STAMP = TABLES_PATH + ".built"  # what it was built for
SOURCES = ("api.cu", "ns_driver.cu", "ns_gemm.cu", "elementwise.cu", "adamw.cu", "profiling.cu", "peer.cu", "no_alloc.cu")
HEADERS = ("common.cuh", "ns_driver.h", "ns_gemm.h", "elementwise.h", "adamw.h", "profiling.h", os.path.join("..", "..", "include", "muon_b200.h"))
TABLES_SOURCES = ("tables.cpp", os.path.join("..", "..", "include", "muon_b200.h"))
NVCC_FLAGS = (
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-lineinfo", "-O3", "-std=c++17",
    "-Xcompiler", "-fPIC",
)


def _nvcc() -> str:
    exe = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(exe):
        raise RuntimeError("nvcc not found: cannot build libmuon_b200.so")
    return exe


def _older(target: str, names) -> bool:
    if not os.path.exists(target):
        return True
    built = os.path.getmtime(target)
    deps = [os.path.join(CSRC, s) for s in names]
    return any(os.path.getmtime(d) > built for d in deps if os.path.exists(d))


def _torch_dir() -> str:
    spec = importlib.util.find_spec("torch")  # the path alone: torch need not be imported to build
    if spec is None or not spec.submodule_search_locations:
        raise RuntimeError("PyTorch not found: cannot build _tables.so")
    return list(spec.submodule_search_locations)[0]


def _tables_target() -> str:
    """The torch and the Python that _tables.so is bound to."""
    return f"torch {importlib.metadata.version('torch')} in {_torch_dir()}, {sys.implementation.cache_tag}\n"


def _tables_stale() -> bool:
    if _older(TABLES_PATH, TABLES_SOURCES) or not os.path.exists(TABLES_STAMP):
        return True
    with open(TABLES_STAMP) as f:
        return f.read() != _tables_target()


def is_stale() -> bool:
    return _older(LIB_PATH, SOURCES + HEADERS) or _tables_stale()


def _run(cmd, verbose: bool = False) -> None:
    if verbose:
        print(" ".join(cmd), file=sys.stderr)
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"{os.path.basename(cmd[0])} failed ({proc.returncode}):\n{proc.stdout}\n{proc.stderr}")
    if verbose:
        print(proc.stderr, file=sys.stderr)


def _build_tables(verbose: bool) -> None:
    torch_dir = _torch_dir()
    include = os.path.join(torch_dir, "include")
    compiler = shutil.which("g++") or shutil.which("c++")
    if compiler is None:
        raise RuntimeError("no C++ compiler found: cannot build _tables.so")
    cuda = os.path.dirname(os.path.dirname(os.path.realpath(_nvcc())))
    # (torch's libraries are loaded already when the extension is; libmuon_b200.so lies beside it)
    _run([compiler, "-O2", "-std=c++17", "-shared", "-fPIC", "-I" + include,
          "-I" + os.path.join(include, "torch", "csrc", "api", "include"),
          "-I" + sysconfig.get_paths()["include"], "-I" + os.path.join(cuda, "include"),
          "-o", TABLES_PATH, os.path.join(CSRC, TABLES_SOURCES[0]),
          "-L" + os.path.join(torch_dir, "lib"), "-ltorch_python", "-ltorch_cpu", "-lc10", "-lc10_cuda",
          "-L" + PKG_DIR, "-lmuon_b200", "-Wl,-rpath,$ORIGIN"], verbose)
    with open(TABLES_STAMP, "w") as f:
        f.write(_tables_target())


def build_library(force: bool = False, verbose: bool = False) -> str:
    """Compile what is missing, older than its sources or made for another torch, files side by side. Returns the
    library's path."""
    jobs = []
    with tempfile.TemporaryDirectory() as tmp, ThreadPoolExecutor() as pool:
        objects = []
        if force or _older(LIB_PATH, SOURCES + HEADERS):
            for name in SOURCES:
                objects.append(os.path.join(tmp, name + ".o"))
                extra = ["-Xptxas", "-v"] if verbose else []
                jobs.append(pool.submit(_run, [_nvcc(), *extra, *NVCC_FLAGS, "-c", "-o", objects[-1],
                                               os.path.join(CSRC, name)], verbose))
        for job in jobs:
            job.result()
        if objects:
            _run([_nvcc(), *NVCC_FLAGS, "-shared", "-o", LIB_PATH, *objects], verbose)
    if force or _tables_stale():
        _build_tables(verbose)
    return LIB_PATH


if __name__ == "__main__":
    print(build_library(force="--force" in sys.argv, verbose="-v" in sys.argv))
