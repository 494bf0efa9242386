"""Build the sm_100a kernel library ``libffa_b200.so`` in-tree with nvcc.

The library is a plain C-ABI shared object (``include/ffa_b200.h``); it is
loaded through ctypes by :mod:`fastest_flash_attention_b200._lib`.  Building
needs only nvcc (cross-compiles without a GPU) and, for the module that calls
it from CPython directly (``csrc/ffa_call.cpp``), g++ and Python's headers.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
import sysconfig
from pathlib import Path

PKG_DIR = Path(__file__).resolve().parent
REPO_DIR = PKG_DIR.parent
CSRC = PKG_DIR / "csrc"
INCLUDE = REPO_DIR / "include"
LIB_NAME = "libffa_b200.so"
LIB_PATH = PKG_DIR / LIB_NAME
CALL_SRC = CSRC / "ffa_call.cpp"
CALL_PATH = PKG_DIR / ("_ffa_call" + sysconfig.get_config_var("EXT_SUFFIX"))
BUILD_DIR = REPO_DIR / "_build"

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-lineinfo", "-std=c++17",
    "-Xcompiler", "-fPIC",
    "--expt-relaxed-constexpr",
]


def _nvcc() -> str:
    cand = os.environ.get("NVCC") or shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not Path(cand).exists() and shutil.which(cand) is None:
        raise RuntimeError("nvcc not found; set NVCC or put CUDA's bin on PATH")
    return cand


def sources() -> list[Path]:
    return sorted(CSRC.glob("*.cu"))


def _stale(obj: Path, src: Path) -> bool:
    if not obj.exists():
        return True
    deps = [src, *CSRC.glob("*.cuh"), *CSRC.glob("*.h"), *INCLUDE.glob("*.h")]
    return any(d.stat().st_mtime > obj.stat().st_mtime for d in deps)


def build_call(verbose: bool = False, force: bool = False) -> Path:
    """Compile ``csrc/ffa_call.cpp``, the CPython side of the C ABI."""
    if force or _stale(CALL_PATH, CALL_SRC):
        tmp = CALL_PATH.with_suffix(".so.tmp")
        cmd = [os.environ.get("CXX") or "g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-Wall", "-I", str(INCLUDE),
               "-I", sysconfig.get_paths()["include"], str(CALL_SRC), "-o", str(tmp)]
        if verbose:
            print(" ".join(cmd), flush=True)
        subprocess.run(cmd, check=True)
        os.replace(tmp, CALL_PATH)
    return CALL_PATH


def build(verbose: bool = False, force: bool = False, jobs: int | None = None) -> Path:
    """Compile every ``csrc/*.cu`` for sm_100a, link ``libffa_b200.so``, and build the module that calls it."""
    nvcc = _nvcc()
    BUILD_DIR.mkdir(exist_ok=True)
    objs = []
    procs = []
    for src in sources():
        obj = BUILD_DIR / (src.stem + ".o")
        objs.append(obj)
        if force or _stale(obj, src):
            cmd = [nvcc, *NVCC_FLAGS, "-I", str(INCLUDE), "-I", str(CSRC), "-c", str(src), "-o", str(obj)]
            if verbose:
                print(" ".join(cmd), flush=True)
            procs.append((src, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT)))
        # bound parallelism
        running = [p for _, p in procs if p.poll() is None]
        while len(running) >= (jobs or os.cpu_count() or 4):
            running[0].wait()
            running = [p for _, p in procs if p.poll() is None]
    for src, p in procs:
        out, _ = p.communicate()
        if p.returncode != 0:
            raise RuntimeError(f"nvcc failed on {src.name}:\n{out.decode(errors='replace')}")
        if verbose and out:
            print(out.decode(errors="replace"))
    if force or not LIB_PATH.exists() or any(o.stat().st_mtime > LIB_PATH.stat().st_mtime for o in objs):
        tmp = LIB_PATH.with_suffix(".so.tmp")
        cmd = [nvcc, "-shared", "-gencode", "arch=compute_100a,code=sm_100a", *map(str, objs), "-o", str(tmp),
               "-lcudart_static", "-ldl", "-lrt", "-lpthread"]
        if verbose:
            print(" ".join(cmd), flush=True)
        subprocess.run(cmd, check=True)
        os.replace(tmp, LIB_PATH)
    build_call(verbose, force)
    return LIB_PATH


if __name__ == "__main__":
    build(verbose="-v" in sys.argv, force="-f" in sys.argv)
    print(LIB_PATH)
