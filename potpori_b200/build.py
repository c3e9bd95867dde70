"""Compile the sm_100a CUDA library in-tree (potpori_b200/libpotpori_b200.so).

nvcc cross-compiles for sm_100a without a GPU. The CUDA runtime is linked statically so the
library does not depend on which libcudart another package (torch) has loaded; the driver
API entry point it needs (tensor-map encoding) is fetched at run time.
"""
from __future__ import annotations

import glob
import os
import shutil
import subprocess
import tempfile
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
LIB = os.path.join(HERE, "libpotpori_b200.so")
SOURCES = [os.path.join(HERE, "csrc", f) for f in (
    "pp_shard.cu", "pp_static_gemv.cu", "pp_prefill.cu", "pp_paged_rows.cu", "pp_tree_attn.cu",
    "pp_tree_tc.cu", "pp_beam.cu")]
DEPS = SOURCES + glob.glob(os.path.join(HERE, "csrc", "*.cuh")) + [
    os.path.join(ROOT, "include", "potpori_b200.h")]

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-lineinfo", "-std=c++17",
    "-Xcompiler", "-fPIC", "-cudart", "static",
    "--expt-relaxed-constexpr",
]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found")


def stale() -> bool:
    if not os.path.exists(LIB):
        return True
    t = os.path.getmtime(LIB)
    return any(os.path.getmtime(p) > t for p in DEPS)


def build(force: bool = False, verbose: bool = False) -> str:
    if not force and not stale():
        return LIB
    env = dict(os.environ)
    env.pop("CC", None)  # the image's CC points at a gcc without the host runtime nvcc wants
    verb = ["-Xptxas=-v"] if verbose else []
    with tempfile.TemporaryDirectory() as tmp:  # the sources side by side, then one link
        objects = [os.path.join(tmp, os.path.basename(s) + ".o") for s in SOURCES]
        jobs = [[nvcc(), *verb, *NVCC_FLAGS, "-c", "-o", o, s] for s, o in zip(SOURCES, objects)]
        with ThreadPoolExecutor(max_workers=os.cpu_count() or 1) as pool:
            list(pool.map(lambda j: subprocess.run(j, check=True, env=env), jobs))
        subprocess.run([nvcc(), *NVCC_FLAGS, "-shared", "-o", LIB + ".tmp", *objects], check=True,
                       env=env)
    os.replace(LIB + ".tmp", LIB)
    return LIB


if __name__ == "__main__":
    import sys
    build(force=True, verbose="-v" in sys.argv)
    print(LIB)
