"""Builds librgb200.so (CUDA kernels + C ABI) in-tree with nvcc for sm_100a.

The arch-specific target has to be spelled as a -gencode pair: the tcgen05 instructions exist only
in the "a" feature set and the shorthand -arch=sm_100a would add a plain compute_100 PTX target
that rejects them.  No fast-math, no FTZ, precise division, no FMA contraction: the output bits are
defined by IEEE single operations (the reference states the same discipline at
repro_gemm_cuda/repro_gemm.cuh:23 and repro_torch/setup.py:24).
"""
import os
import re
import shutil
import subprocess
import time
from concurrent.futures import ThreadPoolExecutor

PKG = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(PKG, "csrc")
LIB = os.path.join(PKG, "librgb200.so")
OBJ = os.path.join(CSRC, "obj")
SOURCES = ["rgb200_api.cu", "rgb200_cxx.cu", "rgb200_optim.cu", "rgb200_norm.cu", "rgb200_epilogue.cu",
           "rgb200_loss.cu", "rgb200_dual.cu"]

NVCC_FLAGS = ["-std=c++17", "-O3", "-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "--fmad=false",
              "-Xcompiler", "-fPIC", "-cudart", "static"]


def _nvcc():
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found; librgb200.so cannot be built")


def _inputs(path, seen=None):
    """The source and every header it includes by a relative path, directly or through another one."""
    seen = set() if seen is None else seen
    path = os.path.normpath(path)
    if path not in seen and os.path.exists(path):
        seen.add(path)
        with open(path) as f:
            for name in re.findall(r'^\s*#include "([^"]+)"', f.read(), re.M):
                _inputs(os.path.join(os.path.dirname(path), name), seen)
    return seen


def _newer(target, inputs):
    return not os.path.exists(target) or any(os.path.getmtime(f) > os.path.getmtime(target) for f in inputs)


def _object(src):
    return os.path.join(OBJ, src[:-3] + ".o")


def stale():
    for src in SOURCES:
        inputs, obj = _inputs(os.path.join(CSRC, src)), _object(src)
        if _newer(LIB, inputs) or (os.path.exists(obj) and _newer(obj, inputs)):
            return True
    return False


def build(force=False, verbose=False):
    """Compile the library if it is missing or older than its sources; returns its path.  Each source becomes an object
    of its own (compiled side by side, reused while its inputs are unchanged), and the objects are linked."""
    if not (force or stale()):
        return LIB
    os.makedirs(OBJ, exist_ok=True)
    nvcc = _nvcc()

    def run(cmd):
        res = subprocess.run(cmd, cwd=CSRC, capture_output=True, text=True)
        if res.returncode != 0:
            raise RuntimeError("nvcc failed:\n" + res.stdout + res.stderr)
        if verbose:
            print(res.stderr)

    def compile_one(src):
        obj = _object(src)
        if force or _newer(obj, _inputs(os.path.join(CSRC, src))):
            began = time.time()
            run([nvcc] + NVCC_FLAGS + (["-Xptxas", "-v"] if verbose else []) + ["-c", "-o", obj, src])
            os.utime(obj, (began, began))       # an input edited while the compiler ran makes the object old
        return obj

    with ThreadPoolExecutor(len(SOURCES)) as pool:
        objs = list(pool.map(compile_one, SOURCES))
    run([nvcc] + NVCC_FLAGS + ["-shared", "-o", LIB] + objs)
    return LIB


if __name__ == "__main__":
    import sys
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
