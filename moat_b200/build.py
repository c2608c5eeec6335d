"""Build recipe for the in-tree CUDA library ``moat_b200/_lib/libmoat_b200.so`` and the
extension module ``moat_bind.so`` beside it (``csrc/bind.cpp``, against the installed torch;
left out where there is none).

Compiles every ``moat_b200/csrc/*.cu`` for sm_100a only (B200), in parallel, and links
one shared library with the C ABI declared in ``include/moat_b200.h``. nvcc
cross-compiles, so this runs on a host without a GPU.

    python -m moat_b200.build          # or __graft_entry__.build()
"""

from __future__ import annotations

import concurrent.futures as cf
import os
import shutil
import subprocess
import sys

PKG = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG)
CSRC = os.path.join(PKG, "csrc")
LIBDIR = os.path.join(PKG, "_lib")
LIB = os.path.join(LIBDIR, "libmoat_b200.so")
BIND = os.path.join(LIBDIR, "moat_bind.so")
OBJDIR = os.path.join(ROOT, "_build", "obj")

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC", "-Xcompiler", "-O3",
         "-I", os.path.join(ROOT, "include")]


def nvcc() -> str:
    for c in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if c and os.path.exists(c):
            return c
    raise RuntimeError("nvcc not found")


def sources() -> list[str]:
    return sorted(os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith(".cu"))


def _compile(src: str, verbose: bool) -> str:
    obj = os.path.join(OBJDIR, os.path.basename(src)[:-3] + ".o")
    cmd = [nvcc(), *ARCH, *FLAGS, "-c", src, "-o", obj]
    if verbose:
        cmd.insert(1, "-Xptxas=-v")
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"nvcc failed on {src}:\n{r.stderr}")
    if verbose and r.stderr:
        sys.stderr.write(r.stderr)
    return obj


def build(verbose: bool = False, force: bool = False) -> str:
    """Compile the CUDA sources into the in-tree shared library, then the binding where torch is
    installed; returns the library's path."""
    build_library(verbose, force)
    build_bind(force)
    return LIB


def build_library(verbose: bool = False, force: bool = False) -> str:
    """Compile the CUDA sources, which need no torch; returns the library's path."""
    srcs = sources()
    deps = srcs + [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith(".cuh")]
    deps.append(os.path.join(ROOT, "include", "moat_b200.h"))
    if not force and os.path.exists(LIB):
        lib_t = os.path.getmtime(LIB)
        if all(os.path.getmtime(d) <= lib_t for d in deps):
            return LIB
    os.makedirs(OBJDIR, exist_ok=True)
    os.makedirs(LIBDIR, exist_ok=True)
    with cf.ThreadPoolExecutor(max_workers=min(8, len(srcs))) as ex:
        objs = list(ex.map(lambda s: _compile(s, verbose), srcs))
    tmp = LIB + ".tmp"
    cmd = [nvcc(), *ARCH, "-shared", "-o", tmp, *objs, "-Xcompiler", "-fPIC"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{r.stderr}")
    os.replace(tmp, LIB)
    return LIB


def build_bind(force: bool = False) -> str | None:
    """Compile the extension module; returns its path, or None where there is no torch."""
    import sysconfig
    try:
        import torch
    except ModuleNotFoundError:
        return None
    src = os.path.join(CSRC, "bind.cpp")
    deps = [src, os.path.join(ROOT, "include", "moat_b200.h"), torch.__file__]
    if not force and os.path.exists(BIND) and all(os.path.getmtime(d) <= os.path.getmtime(BIND) for d in deps):
        return BIND
    os.makedirs(LIBDIR, exist_ok=True)
    home = os.path.dirname(torch.__file__)
    cuda = os.path.dirname(os.path.dirname(nvcc()))
    tmp = BIND + ".tmp"
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}", "-I", os.path.join(ROOT, "include"),
           "-I", os.path.join(home, "include"), "-I", sysconfig.get_paths()["include"],
           "-I", os.path.join(cuda, "include"), src, "-o", tmp, "-L", os.path.join(home, "lib"), "-ltorch_python",
           "-ltorch_cpu", "-lc10", "-lc10_cuda"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"{cmd[0]} failed on {src}:\n{r.stderr}")
    os.replace(tmp, BIND)
    return BIND


if __name__ == "__main__":
    print(build(verbose="-v" in sys.argv, force="-f" in sys.argv))
