"""In-tree build of librocm_dev_b200.so (hand-written CUDA for sm_100a).

nvcc cross-compiles without a GPU.  The shared object lands next to this file
so that it travels with the source tree; it links the CUDA runtime statically
and resolves the driver lazily, so it also loads on a machine with no GPU.
"""
from __future__ import annotations

import glob
import os
import subprocess
import sysconfig

_HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(_HERE, "csrc")
LIB_PATH = os.path.join(_HERE, "librocm_dev_b200.so")
FAST_PATH = os.path.join(_HERE, "_fastcall.so")     # optional: see csrc/fastcall.c

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-lineinfo", "-O3", "-std=c++17",
    "-shared", "-Xcompiler", "-fPIC",
    "--cudart", "static",
]


def sources() -> list[str]:
    return sorted(glob.glob(os.path.join(CSRC, "*.cu")))


def _stale() -> bool:
    if not os.path.exists(LIB_PATH):
        return True
    t = os.path.getmtime(LIB_PATH)
    deps = sources() + glob.glob(os.path.join(CSRC, "*.cuh")) + glob.glob(os.path.join(CSRC, "*.h")) + glob.glob(os.path.join(CSRC, "*.c"))
    deps.append(os.path.join(_HERE, "..", "include", "rocm_dev_b200.h"))
    return any(os.path.getmtime(d) > t for d in deps)


def build(force: bool = False, verbose: bool = False) -> str:
    """Compile every kernel source into one shared library; returns its path."""
    if not force and not _stale():
        return LIB_PATH
    nvcc = os.environ.get("NVCC", "nvcc")
    cmd = [nvcc, *NVCC_FLAGS]
    if verbose:
        cmd += ["-Xptxas", "-v"]
    cmd += ["-o", LIB_PATH, *sources()]
    subprocess.check_call(cmd)
    _build_fastcall()
    return LIB_PATH


def _build_fastcall() -> None:
    """The C entry of the short calls, where the Python headers are there; without it ctypes does the same."""
    include = sysconfig.get_paths()["include"]
    if os.path.exists(FAST_PATH):
        os.remove(FAST_PATH)
    if os.path.exists(os.path.join(include, "Python.h")):
        subprocess.check_call([os.environ.get("CC", "gcc"), "-O2", "-shared", "-fPIC", "-I", include, "-o", FAST_PATH,
                               os.path.join(CSRC, "fastcall.c")])


if __name__ == "__main__":
    print(build(force=True, verbose=True))
