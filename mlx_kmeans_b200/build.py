"""Compile the CUDA library libkmc.so in-tree (sm_100a) from csrc/*.cu, and on top of it the module _experts (torch
tensors to the routed-experts entry points, csrc/bind_experts.cpp).

    python -m mlx_kmeans_b200.build          # or: python mlx_kmeans_b200/build.py

nvcc cross-compiles without a GPU, so this runs on any machine with the CUDA 12.9 toolkit (without torch, libkmc.so
alone is built).  Objects are
compiled in parallel and relinked only when a source or header is newer than the library.
"""
import concurrent.futures
import glob
import os
import shutil
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
OBJ = os.path.join(HERE, "_build")
LIB = os.path.join(HERE, "libkmc.so")
BIND_SRC = os.path.join(CSRC, "bind_experts.cpp")
BIND = os.path.join(HERE, "_experts.so")

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC", "--expt-relaxed-constexpr",
         "-I" + os.path.join(ROOT, "include")]


def nvcc():
    exe = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(exe):
        raise RuntimeError("nvcc not found: the CUDA toolkit is needed to build libkmc.so")
    return exe


def _sources():
    return sorted(glob.glob(os.path.join(CSRC, "*.cu")))


def _deps():
    return (sorted(glob.glob(os.path.join(CSRC, "*.cu*"))) + sorted(glob.glob(os.path.join(CSRC, "*.h")))
            + [os.path.join(ROOT, "include", "kmc.h")])


def up_to_date():
    if not os.path.exists(LIB):
        return False
    t = os.path.getmtime(LIB)
    return all(os.path.getmtime(p) <= t for p in _deps())


def build(verbose=False, force=False, extra=()):
    """Compile every csrc/*.cu for sm_100a and link libkmc.so (static cudart). Returns the library path."""
    if not force and not extra and up_to_date():
        build_binding(verbose, force)
        return LIB
    os.makedirs(OBJ, exist_ok=True)
    exe = nvcc()
    srcs = _sources()

    def compile_one(src):
        obj = os.path.join(OBJ, os.path.basename(src)[:-3] + ".o")
        cmd = [exe] + ARCH + FLAGS + list(extra) + ["-c", src, "-o", obj]
        if verbose:
            print(" ".join(cmd), flush=True)
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"nvcc failed on {os.path.basename(src)}:\n{r.stdout}\n{r.stderr}")
        if verbose and (r.stdout or r.stderr):
            print(r.stdout + r.stderr, flush=True)
        return obj

    with concurrent.futures.ThreadPoolExecutor(max_workers=min(8, len(srcs))) as pool:
        objs = list(pool.map(compile_one, srcs))
    tmp = LIB + ".tmp"
    cmd = [exe] + ARCH + ["-shared", "-o", tmp] + objs
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link of libkmc.so failed:\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, LIB)
    build_binding(verbose, force)
    return LIB


def build_binding(verbose=False, force=False):
    """Compile csrc/bind_experts.cpp against the installed torch and link it to libkmc.so. Returns its path, or None on a
    machine without torch, where libkmc.so alone is of use."""
    deps = [BIND_SRC, os.path.join(ROOT, "include", "kmc.h")]
    if not force and os.path.exists(BIND) and all(os.path.getmtime(p) <= os.path.getmtime(BIND) for p in deps):
        return BIND
    try:
        import torch
    except ImportError:
        print("torch is not installed: the module _experts is not built", file=sys.stderr)
        return None
    base = os.path.dirname(torch.__file__)
    inc = [os.path.join(base, "include"), os.path.join(base, "include", "torch", "csrc", "api", "include"),
           os.path.join(os.path.dirname(os.path.dirname(nvcc())), "include"), sysconfig.get_paths()["include"]]
    tmp = BIND + ".tmp"
    cmd = [shutil.which("g++") or "g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-DTORCH_EXTENSION_NAME=_experts",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}"]
    cmd += [a for i in inc for a in ("-isystem", i)] + [BIND_SRC, "-o", tmp, "-L" + HERE, "-l:libkmc.so"]
    cmd += ["-L" + os.path.join(base, "lib"), "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_cuda", "-ltorch",
            "-ltorch_python", "-Wl,-rpath,$ORIGIN"]
    if verbose:
        print(" ".join(cmd), flush=True)
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"g++ failed on bind_experts.cpp:\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, BIND)
    return BIND


if __name__ == "__main__":
    print(build(verbose="-v" in sys.argv, force="-f" in sys.argv))
