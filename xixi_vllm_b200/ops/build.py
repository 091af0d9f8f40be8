"""Builds the sm_100a kernel library in-tree with nvcc (cross-compiles without a GPU).

    python -m xixi_vllm_b200.ops.build [--force] [--verbose]

Produces ``xixi_vllm_b200/ops/_xv_cuda.so``; the source list is every ``.cu`` under
``csrc/kernels``. The shared object carries only sm_100a code: there is no fallback arch.
``build_torch`` produces ``_xv_torch.so`` with g++: the Python calls of the 4-bit cache operators
(``csrc/host/kv4_torch.cpp``), compiled against the installed torch.
"""

from __future__ import annotations

import argparse
import glob
import os
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

_HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(os.path.dirname(_HERE), "csrc")
LIB = os.path.join(_HERE, "_xv_cuda.so")
OBJ_DIR = os.path.join(_HERE, "_build")
TORCH_SRC = os.path.join(CSRC, "host", "kv4_torch.cpp")
TORCH_LIB = os.path.join(_HERE, "_xv_torch.so")

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17",
    "--use_fast_math", "-Xcompiler", "-fPIC", "--expt-relaxed-constexpr",
]


def nvcc_path() -> str:
    p = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(p):
        raise FileNotFoundError("nvcc not found")
    return p


def sources() -> list[str]:
    return sorted(glob.glob(os.path.join(CSRC, "kernels", "*.cu")))


def _headers() -> list[str]:
    return (glob.glob(os.path.join(CSRC, "common", "*.cuh")) + glob.glob(os.path.join(CSRC, "kernels", "*.cuh"))
            + glob.glob(os.path.join(CSRC, "kernels", "*.h")))


def _deps_mtime() -> float:
    files = sources() + _headers()
    return max(os.path.getmtime(f) for f in files)


def needs_build() -> bool:
    return not os.path.isfile(LIB) or os.path.getmtime(LIB) < _deps_mtime()


def build(force: bool = False, verbose: bool = False) -> str:
    if not force and not needs_build():
        return LIB
    nvcc = nvcc_path()
    os.makedirs(OBJ_DIR, exist_ok=True)
    extra = ["-Xptxas", "-v"] if verbose else []
    hdr_time = max([os.path.getmtime(f) for f in _headers()] or [0.0])

    def compile_one(src: str) -> str:
        obj = os.path.join(OBJ_DIR, os.path.basename(src)[:-3] + ".o")
        if not force and os.path.isfile(obj) and os.path.getmtime(obj) >= max(os.path.getmtime(src), hdr_time):
            return obj
        cmd = [nvcc, *NVCC_FLAGS, *extra, "-I", os.path.join(CSRC, "kernels"), "-c", src, "-o", obj]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if verbose or r.returncode:
            sys.stderr.write(r.stdout + r.stderr)
        if r.returncode:
            raise RuntimeError(f"nvcc failed for {src}")
        return obj

    with ThreadPoolExecutor(max_workers=min(8, os.cpu_count() or 1)) as ex:
        objs = list(ex.map(compile_one, sources()))
    tmp = LIB + f".tmp{os.getpid()}"
    subprocess.run([nvcc, "-shared", "-o", tmp, *objs], check=True)
    os.replace(tmp, LIB)
    return LIB


def _built_for() -> str:
    """What a Python extension fits: it is compiled against one torch and one Python."""
    import torch

    return f"xv built for torch {torch.__version__} {sys.implementation.cache_tag};"


def _torch_lib_fits() -> bool:
    """The extension is there, no older than its sources, and carries the mark of this torch and Python."""
    header = os.path.join(CSRC, "kernels", "xv_cuda.h")
    if not os.path.isfile(TORCH_LIB) or os.path.getmtime(TORCH_LIB) < max(map(os.path.getmtime, (TORCH_SRC, header))):
        return False
    with open(TORCH_LIB, "rb") as f:
        return _built_for().encode() in f.read()


def build_torch(force: bool = False) -> str:
    """Compile the Python extension in-tree with g++ (half a minute: torch's headers)."""
    if not force and _torch_lib_fits():
        return TORCH_LIB
    import sysconfig

    import torch

    root = os.path.dirname(torch.__file__)
    cuda = os.path.dirname(os.path.dirname(os.path.realpath(nvcc_path())))
    tmp = TORCH_LIB + f".tmp{os.getpid()}"
    subprocess.run(["g++", "-O2", "-std=c++17", "-shared", "-fPIC", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}",
                    f'-DXV_BUILT_FOR="{_built_for()}"',
                    "-isystem", os.path.join(root, "include"),
                    "-isystem", os.path.join(root, "include", "torch", "csrc", "api", "include"),
                    "-isystem", os.path.join(cuda, "include"), "-isystem", sysconfig.get_paths()["include"],
                    "-I", os.path.join(CSRC, "kernels"), "-o", tmp, TORCH_SRC,
                    "-L", os.path.join(root, "lib"), "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_cuda", "-ltorch_python"], check=True)
    os.replace(tmp, TORCH_LIB)
    return TORCH_LIB


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--verbose", action="store_true")
    a = ap.parse_args()
    print(build(a.force, a.verbose))
    print(build_torch(a.force))
