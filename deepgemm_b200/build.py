"""Ahead-of-time build of libmegamoe_b200.so with nvcc for sm_100a (no JIT, no CUTLASS).

    python -m deepgemm_b200.build [--force] [--verbose]

The shared object is written next to this file so that it is found by deepgemm_b200._lib and
travels with the source tree.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB_NAME = "libmegamoe_b200.so"
LIB_PATH = os.path.join(HERE, LIB_NAME)
SOURCES = ["abi.cu", "noalloc.cu", "block128.cu"]
HEADERS = ["layout.h", "pack.cuh", "ptx.cuh", "route.cuh", "gemm.cuh", "gemm_pair.cuh", "gemm_ue8m0.cuh", "misc.cuh", "deepep_layout.cuh", "split_baseline.cuh", "fused.cuh", "probe.cuh", "block128.cuh", "block128_gemm.cuh", "block128_moe.cuh",
           os.path.join("..", "..", "include", "megamoe_b200.h")]


def _nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found; set NVCC or put it on PATH")


def needs_build() -> bool:
    if not os.path.exists(LIB_PATH):
        return True
    t = os.path.getmtime(LIB_PATH)
    deps = [os.path.join(CSRC, s) for s in SOURCES] + [os.path.join(CSRC, h) for h in HEADERS] + [__file__]
    return any(os.path.exists(d) and os.path.getmtime(d) > t for d in deps)


def build(force: bool = False, verbose: bool = False) -> str:
    if not force and not needs_build():
        return LIB_PATH
    cmd = [_nvcc(), "-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17",
           "-shared", "-Xcompiler", "-fPIC",
           "-o", LIB_PATH] + [os.path.join(CSRC, s) for s in SOURCES]
    if verbose:
        cmd.insert(1, "-Xptxas")
        cmd.insert(2, "-v")
        print(" ".join(cmd), flush=True)
    res = subprocess.run(cmd, capture_output=True, text=True)
    if verbose or res.returncode != 0:
        sys.stderr.write(res.stdout + res.stderr)
    if res.returncode != 0:
        raise RuntimeError("nvcc failed building " + LIB_NAME)
    return LIB_PATH


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="--verbose" in sys.argv))
