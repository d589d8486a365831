"""Build libmgprims.so (the HIP kernels + C ABI) in-tree for gfx950.

    python muse-glimmer-intel-serve_amd/build.py

Every source compiles with hipcc for gfx950 only, with FP contraction off (the
bitwise contract with the reference depends on unfused multiply/add, as the
reference's own -ffp-contract=off does, CMakeLists.txt:11-14), without
fast-math, and with packed-f32 instruction selection disabled.
"""
from __future__ import annotations

import concurrent.futures as cf
import os
import shutil
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libmgprims.so")
OBJ = os.path.join(HERE, "_build")
ARCH = "gfx950"

SOURCES = ["mg_api.cpp", "mg_npy.cpp", "k_norm.hip", "k_elementwise.hip", "k_rope.hip", "k_qk.hip", "k_softmax.hip", "k_softmax64.hip",
           "k_q8.hip", "k_vocab.hip", "k_sample.hip", "k_attn.hip", "k_attn_prefill.hip", "k_pages.hip",
           "k_attn_paged.hip", "k_mxfp4.hip", "k_mxfp4_gemv.hip", "k_mxfp4_gemm.hip", "k_attn_mxfp4.hip", "k_probe.hip"]

FLAGS = [
    "-x", "hip", f"--offload-arch={ARCH}", "-O3", "-fPIC", "-std=c++17",
    "-ffp-contract=off", "-fno-fast-math", "-fno-gpu-flush-denormals-to-zero",
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-Wall", "-Wno-unused-function",
    f"-I{os.path.join(ROOT, 'include')}", f"-I{CSRC}",
]


def hipcc() -> str:
    for c in (os.environ.get("HIPCC"), "/opt/rocm/bin/hipcc", shutil.which("hipcc")):
        if c and os.path.exists(c):
            return c
    raise RuntimeError("hipcc not found")


def _compile(src: str) -> str:
    obj = os.path.join(OBJ, os.path.splitext(src)[0] + ".o")
    cmd = [hipcc(), *FLAGS, "-c", os.path.join(CSRC, src), "-o", obj]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"compile failed: {src}\n{' '.join(cmd)}\n{r.stdout}\n{r.stderr}")
    return obj


def build(verbose: bool = True) -> str:
    os.makedirs(OBJ, exist_ok=True)
    jobs = min(len(SOURCES), max(1, (os.cpu_count() or 4)))
    with cf.ThreadPoolExecutor(jobs) as ex:
        objs = list(ex.map(_compile, SOURCES))
    tmp = LIB + ".tmp"
    cmd = [hipcc(), f"--offload-arch={ARCH}", "-shared", "-fPIC", "-o", tmp, *objs]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed\n{' '.join(cmd)}\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, LIB)
    if verbose:
        print(f"built {LIB}")
    return LIB


if __name__ == "__main__":
    try:
        build()
    except RuntimeError as e:
        print(e, file=sys.stderr)
        sys.exit(1)
