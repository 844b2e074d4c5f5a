#!/usr/bin/env python3
"""Builds libvoxq.so (all CUDA sources for sm_100a) next to this file and, where PyTorch is installed, the binding of
the batched operators to torch tensors (csrc/voxq_torch.cpp) as voxq/_torch.so.  A C user needs nvcc alone.

    python voxcpm2-c_b200/build.py [-j N] [--force]

Objects go to _build/ (git-ignored); the shared library lands in this folder so
it travels with the repository snapshot.  Each .cu is recompiled when it or any
header under csrc/ or include/ is newer than its object.
"""
from __future__ import annotations

import argparse
import concurrent.futures as cf
import glob
import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
REPO = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
OBJ = os.path.join(HERE, "_build")
LIB = os.path.join(HERE, "libvoxq.so")
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")

FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-lineinfo", "-O3", "-std=c++17",
    "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=hidden",
    "--expt-relaxed-constexpr",
    "-I", os.path.join(REPO, "include"), "-I", CSRC,
]


def _headers_mtime() -> float:
    hs = glob.glob(os.path.join(CSRC, "*.h")) + glob.glob(os.path.join(CSRC, "*.cuh")) + \
        glob.glob(os.path.join(REPO, "include", "*.h"))
    return max((os.path.getmtime(h) for h in hs), default=0.0)


def _compile(src: str, force: bool, verbose: bool) -> str:
    obj = os.path.join(OBJ, os.path.basename(src)[:-3] + ".o")
    if not force and os.path.exists(obj):
        t = os.path.getmtime(obj)
        if t >= os.path.getmtime(src) and t >= _headers_mtime():
            return obj
    cmd = [NVCC, *FLAGS, "-c", src, "-o", obj]
    if verbose:
        cmd.insert(1, "-Xptxas=-v")
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        sys.stderr.write(r.stdout + r.stderr)
        raise RuntimeError(f"nvcc failed on {src}")
    if verbose:
        sys.stderr.write(r.stderr)
    return obj


def build(force: bool = False, jobs: int = 8, verbose: bool = False) -> str:
    os.makedirs(OBJ, exist_ok=True)
    srcs = sorted(glob.glob(os.path.join(CSRC, "*.cu")))
    with cf.ThreadPoolExecutor(max_workers=jobs) as ex:
        objs = list(ex.map(lambda s: _compile(s, force, verbose), srcs))
    if force or not os.path.exists(LIB) or max(os.path.getmtime(o) for o in objs) > os.path.getmtime(LIB):
        cmd = [NVCC, "-gencode", "arch=compute_100a,code=sm_100a", "-shared", "-o", LIB, *objs, "-lcuda"]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            sys.stderr.write(r.stdout + r.stderr)
            raise RuntimeError("link failed")
    build_binding(force)
    return LIB


def build_binding(force: bool = False) -> str | None:
    """voxq/_torch.so: a CPython module against the installed torch's headers and libraries; rebuilt when its source or
    either of them changes.  Without PyTorch there is nothing to bind: returns None."""
    import sysconfig
    try:
        import torch
    except ImportError:
        sys.stderr.write("no PyTorch: voxq/_torch.so (the batched operators on torch tensors) is not built\n")
        return None
    src, out = os.path.join(CSRC, "voxq_torch.cpp"), os.path.join(HERE, "voxq", "_torch.so")
    header = os.path.join(REPO, "include", "voxq.h")
    stamp, made = os.path.join(OBJ, "_torch.stamp"), f"torch {torch.__version__} at {torch.__file__}, Python {sys.version}\n"
    if not force and os.path.exists(out) and os.path.exists(stamp) and open(stamp).read() == made and \
            os.path.getmtime(out) > max(os.path.getmtime(src), os.path.getmtime(header)):
        return out
    root = os.path.dirname(torch.__file__)
    lib, inc = os.path.join(root, "lib"), os.path.join(root, "include")
    cuda = os.path.join(os.path.dirname(os.path.dirname(NVCC)), "include")
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden", "-w", src, "-o", out,
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", "-I", os.path.join(REPO, "include"),
           "-I", cuda, "-I", sysconfig.get_paths()["include"], "-I", inc, "-I", os.path.join(inc, "torch", "csrc", "api", "include"),
           "-L", lib, "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_cuda", "-ltorch_python", f"-Wl,-rpath,{lib}"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        sys.stderr.write(r.stdout + r.stderr)
        raise RuntimeError(f"g++ failed on {src}")
    os.makedirs(OBJ, exist_ok=True)
    with open(stamp, "w") as f:
        f.write(made)
    return out


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("-j", type=int, default=8)
    ap.add_argument("--force", action="store_true")
    ap.add_argument("-v", "--verbose", action="store_true", help="print ptxas register/spill stats")
    a = ap.parse_args()
    print(build(a.force, a.j, a.verbose))
