"""Compile the sm_100a CUDA library in-tree (potpori_b200/libpotpori_b200.so) and its torch binding
(potpori_b200/_paged.so). The binding alone needs torch and a host compiler: where torch is not installed,
the library is built and the binding left out.

nvcc cross-compiles for sm_100a without a GPU. The CUDA runtime is linked statically so the
library does not depend on which libcudart another package (torch) has loaded; the driver
API entry point it needs (tensor-map encoding) is fetched at run time.
"""
from __future__ import annotations

import glob
import importlib.metadata
import importlib.util
import os
import shutil
import subprocess
import sys
import sysconfig
import tempfile
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
LIB = os.path.join(HERE, "libpotpori_b200.so")
SOURCES = [os.path.join(HERE, "csrc", f) for f in (
    "pp_shard.cu", "pp_static_gemv.cu", "pp_prefill.cu", "pp_paged_rows.cu", "pp_tree_attn.cu",
    "pp_tree_tc.cu", "pp_beam.cu")]
HEADER = os.path.join(ROOT, "include", "potpori_b200.h")
DEPS = SOURCES + glob.glob(os.path.join(HERE, "csrc", "*.cuh")) + [HEADER]
BINDING = os.path.join(HERE, "_paged.so")
BINDING_SOURCE = os.path.join(HERE, "csrc", "pp_torch.cpp")
BINDING_BUILT_FOR = os.path.join(HERE, "_paged.built")  # the torch and Python that _paged.so was built for

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


def stale(target: str = LIB, deps: list = DEPS) -> bool:
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(p) > t for p in deps)


def binding_abi() -> "str | None":
    """The torch and Python that a binding is built for; None without torch."""
    if importlib.util.find_spec("torch") is None:
        return None
    try:
        version = importlib.metadata.version("torch")
    except importlib.metadata.PackageNotFoundError:  # a source tree on the path
        import torch
        version = torch.__version__
    return f"torch {version} {sysconfig.get_config_var('SOABI')}"


def binding_stale(abi: str) -> bool:
    """Older than its sources, or built for another torch or Python, whose C++ ABI may differ."""
    if stale(BINDING, [BINDING_SOURCE, HEADER]) or not os.path.exists(BINDING_BUILT_FOR):
        return True
    with open(BINDING_BUILT_FOR) as f:
        return f.read() != abi


def build_binding(abi: str) -> None:
    """potpori_b200/_paged.so: the paged operators' torch binding, linked to the library beside it."""
    from torch.utils import cpp_extension

    cxx = next((c for c in ("/usr/bin/g++", shutil.which("g++")) if c and os.path.exists(c)), "c++")
    torch_lib = cpp_extension.library_paths()[0]
    includes = cpp_extension.include_paths() + ["/usr/local/cuda/include", sysconfig.get_paths()["include"]]
    subprocess.run(
        [cxx, "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden", BINDING_SOURCE, "-o", BINDING + ".tmp",
         *(f"-isystem{p}" for p in includes), f"-L{torch_lib}", "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch",
         "-ltorch_python", f"-L{HERE}", "-l:" + os.path.basename(LIB), "-Wl,-rpath,$ORIGIN",
         f"-Wl,-rpath,{torch_lib}"], check=True)
    os.replace(BINDING + ".tmp", BINDING)
    with open(BINDING_BUILT_FOR, "w") as f:
        f.write(abi)


def build(force: bool = False, verbose: bool = False) -> str:
    if force or stale():
        build_library(verbose)
    abi = binding_abi()
    if abi is None:
        print("torch is not installed: potpori_b200.paged is left out", file=sys.stderr)
    elif force or binding_stale(abi):
        build_binding(abi)
    return LIB


def build_library(verbose: bool = False) -> None:
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


if __name__ == "__main__":
    build(force=True, verbose="-v" in sys.argv)
    print(LIB)
