"""Build libpam_cuda.so (the C-ABI CUDA library) in-tree with nvcc for sm_100a.

    python -m pagedattentionmetal_b200.build [--force] [--verbose]

Objects go to pagedattentionmetal_b200/build/, the library next to this file.
nvcc cross-compiles without a GPU.
"""
from __future__ import annotations

import concurrent.futures as cf
import os
import shutil
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OBJ = os.path.join(HERE, "build")
LIB = os.path.join(HERE, "libpam_cuda.so")
INCLUDE = os.path.join(HERE, "..", "include")

SOURCES = ["cache_kernels.cu", "decode_kernels.cu", "decode_stream_kernel.cu", "prefill_kernels.cu", "prefill_tc_kernel.cu", "backward_kernels.cu", "backward_mma_kernels.cu", "pam_cabi.cu",
           "comm.cu", "step_kernels.cu", "norm_rotate_kernels.cu", "tree_kernels.cu", "tree_mma_kernel.cu", "tree_tc_kernel.cu", "block_manager.cpp"]
HEADERS = ["kernels.h", "step_calls.inl", "tree_common.cuh", "tc_common.cuh", "block_manager.h", os.path.join(INCLUDE, "pam_cuda.h")]

NVCC_FLAGS = [
    "-O3", "-std=c++17", "-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo",
    "-Xcompiler", "-fPIC", "-Xcompiler", "-Wall", "--expt-relaxed-constexpr",
]


def nvcc() -> str:
    exe = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(exe):
        raise RuntimeError("nvcc not found; the CUDA toolkit is required to build libpam_cuda.so")
    return exe


def _newest_input() -> float:
    paths = [os.path.join(CSRC, s) for s in SOURCES]
    paths += [h if os.path.isabs(h) else os.path.join(CSRC, h) for h in HEADERS]
    return max(os.path.getmtime(p) for p in paths)


def up_to_date() -> bool:
    return os.path.exists(LIB) and os.path.getmtime(LIB) >= _newest_input()


def build(force: bool = False, verbose: bool = False) -> str:
    if not force and up_to_date():
        return LIB
    os.makedirs(OBJ, exist_ok=True)
    cc = nvcc()

    def compile_one(src: str) -> str:
        obj = os.path.join(OBJ, os.path.splitext(src)[0] + ".o")
        cmd = [cc, *NVCC_FLAGS, "-I", INCLUDE, "-c", os.path.join(CSRC, src), "-o", obj]
        if verbose:
            cmd.insert(1, "-Xptxas")
            cmd.insert(2, "-v")
        r = subprocess.run(cmd, capture_output=True, text=True)
        if verbose or r.returncode != 0:
            sys.stderr.write(r.stdout + r.stderr)
        if r.returncode != 0:
            raise RuntimeError(f"nvcc failed on {src}")
        return obj

    with cf.ThreadPoolExecutor(max_workers=len(SOURCES)) as ex:
        objs = list(ex.map(compile_one, SOURCES))
    cmd = [cc, "-shared", "-o", LIB, *objs, "-gencode", "arch=compute_100a,code=sm_100a"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        sys.stderr.write(r.stdout + r.stderr)
        raise RuntimeError("link of libpam_cuda.so failed")
    return LIB


if __name__ == "__main__":
    path = build(force="--force" in sys.argv, verbose="--verbose" in sys.argv)
    print(path)
