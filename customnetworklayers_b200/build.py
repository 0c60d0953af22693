"""Builds the C-ABI shared library in-tree with nvcc for sm_100a (cross-compiles without a GPU).

    python -m customnetworklayers_b200.build [--force] [--verbose]
"""
from __future__ import annotations

import os
import subprocess
import sys
import tempfile
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB_PATH = os.path.join(HERE, "libcnl_b200.so")
SOURCES = ["common.cu", "tv_fista.cu", "tv_fused.cu", "tv_flow.cu", "peer_allreduce.cu", "tv_noalloc.cu", "median.cu", "quadfit.cu", "tgv.cu", "tgv_vec.cu", "wmedian.cu",
           "ckpt8.cu", "blocknorm.cu", "blocknorm_vec.cu", "linattn.cu", "linattn_f32.cu", "linattn_mma.cu",
           "linattn_tc.cu"]
HEADERS = ["common.h", "tv_math.cuh", "tv_fused.cuh", "tv_tile.cuh", "tgv_vec.cuh", "dtypes.cuh", "ckpt8.cuh", "blocknorm.cuh", "linattn.cuh",
           os.path.join("..", "..", "include", "cnl_b200.h")]
NVCC_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17",
              "-Xcompiler", "-fPIC", "--cudart", "shared"]


def _nvcc() -> str:
    for cand in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", "nvcc"):
        if cand and (os.path.isabs(cand) and os.path.exists(cand) or not os.path.isabs(cand)):
            return cand
    return "nvcc"


def needs_build() -> bool:
    if not os.path.exists(LIB_PATH):
        return True
    t = os.path.getmtime(LIB_PATH)
    deps = [os.path.join(CSRC, s) for s in SOURCES + HEADERS] + [os.path.abspath(__file__)]
    return any(os.path.getmtime(d) > t for d in deps if os.path.exists(d))


def build(force: bool = False, verbose: bool = False) -> str:
    """Compiles every .cu of the package into libcnl_b200.so; returns the library path."""
    if not force and not needs_build():
        return LIB_PATH
    flags = NVCC_FLAGS + (["-Xptxas", "-v"] if verbose else [])
    with tempfile.TemporaryDirectory() as tmp:                    # every source on its own, as many at a time as there are cores
        objects = [os.path.join(tmp, s + ".o") for s in SOURCES]
        cmds = [[_nvcc()] + flags + ["-c", os.path.join(CSRC, s), "-o", o] for s, o in zip(SOURCES, objects)]
        with ThreadPoolExecutor(max(1, os.cpu_count() or 1)) as pool:
            results = list(pool.map(lambda c: subprocess.run(c, capture_output=True, text=True), cmds))
        if all(r.returncode == 0 for r in results):
            results.append(subprocess.run([_nvcc()] + NVCC_FLAGS + ["-shared"] + objects + ["-o", LIB_PATH], capture_output=True, text=True))
    failed = [r for r in results if r.returncode != 0]
    for res in results if verbose else failed:
        sys.stderr.write(res.stdout + res.stderr)
    if failed:
        raise RuntimeError("nvcc failed building libcnl_b200.so")
    return LIB_PATH


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="--verbose" in sys.argv))
