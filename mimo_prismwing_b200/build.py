"""Build the sm_100a CUDA library behind include/pw_cuda.h.

Compiles every mimo_prismwing_b200/csrc/*.cu for sm_100a, and the host-only
csrc/*.cpp (checkpoint ingestion) with the same driver (`-gencode
arch=compute_100a,code=sm_100a -lineinfo`, no fast-math: the quantizer and the
staged SwiGLU rely on IEEE division and rounding) and links
mimo_prismwing_b200/lib/libpw_cuda.so in-tree, and compiles the binding for torch
tensors (binding/pw_torch.cpp) with g++ to mimo_prismwing_b200/lib/, one file per
version of torch and Python.
Objects go to mimo_prismwing_b200/_build/ (not committed).
"""
from __future__ import annotations

import concurrent.futures as cf
import glob
import importlib.util
import os
import subprocess
import sys
import sysconfig

from ._lib import BINDING_PATH

PKG = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG)
CSRC = os.path.join(PKG, "csrc")
BUILD = os.path.join(PKG, "_build")
LIB = os.path.join(PKG, "lib", "libpw_cuda.so")
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC", "-I" + os.path.join(ROOT, "include"),
         "-I" + CSRC]


def _stale(target: str, deps: list[str]) -> bool:
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


def build_binding(force: bool = False) -> None:
    """The Python extension over torch's and the library's headers."""
    src = os.path.join(PKG, "binding", "pw_torch.cpp")
    if not force and not _stale(BINDING_PATH, [src] + glob.glob(os.path.join(ROOT, "include", "*.h"))):
        return
    torch = importlib.util.find_spec("torch").submodule_search_locations[0]
    include = [os.path.join(ROOT, "include"), os.path.join(torch, "include"),
               os.path.join(torch, "include", "torch", "csrc", "api", "include"), sysconfig.get_paths()["include"]]
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-shared", "-fPIC", "-fvisibility=hidden"]
    cmd += ["-I" + d for d in include] + [src, "-o", BINDING_PATH, "-L" + os.path.join(torch, "lib")]
    res = subprocess.run(cmd + ["-ltorch_python", "-ltorch_cpu", "-lc10"], capture_output=True, text=True)
    if res.returncode != 0:
        sys.stderr.write(res.stdout + res.stderr)
        raise RuntimeError("the binding did not build")


def build(verbose: bool = False, force: bool = False) -> str:
    os.makedirs(BUILD, exist_ok=True)
    os.makedirs(os.path.dirname(LIB), exist_ok=True)
    sources = sorted(glob.glob(os.path.join(CSRC, "*.cu")) + glob.glob(os.path.join(CSRC, "*.cpp")))
    headers = glob.glob(os.path.join(CSRC, "*.h")) + glob.glob(os.path.join(CSRC, "*.cuh")) + \
        glob.glob(os.path.join(ROOT, "include", "*.h"))
    objects = []
    jobs = []
    for src in sources:
        obj = os.path.join(BUILD, os.path.splitext(os.path.basename(src))[0] + ".o")
        objects.append(obj)
        if force or _stale(obj, [src] + headers):
            cmd = [NVCC] + ARCH + FLAGS + ["-c", src, "-o", obj]
            if verbose:
                cmd.insert(1, "-Xptxas=-v")
            jobs.append(cmd)
    with cf.ThreadPoolExecutor(max_workers=max(1, min(8, os.cpu_count() or 1))) as ex:
        for cmd, res in zip(jobs, ex.map(lambda c: subprocess.run(c, capture_output=True, text=True), jobs)):
            if verbose or res.returncode != 0:
                sys.stderr.write(res.stdout + res.stderr)
            if res.returncode != 0:
                raise RuntimeError("nvcc failed: " + " ".join(cmd))
    if force or jobs or _stale(LIB, objects):
        cmd = [NVCC] + ARCH + ["-shared", "-o", LIB] + objects + ["-lcudart_static", "-lrt", "-ldl", "-lpthread"]
        res = subprocess.run(cmd, capture_output=True, text=True)
        if res.returncode != 0:
            sys.stderr.write(res.stdout + res.stderr)
            raise RuntimeError("link failed")
    build_binding(force)
    return LIB


if __name__ == "__main__":
    print(build(verbose="-v" in sys.argv, force="-f" in sys.argv))
