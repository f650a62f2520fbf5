"""Builds ``libdyllm_b200.so`` in-tree with nvcc for sm_100a, and ``_native.so``, the Python binding of the entry points on
8-bit caches, with the C++ compiler against torch's headers.

Usage: ``python -m dyllm_b200.build [--force] [--verbose]``.  The library has no torch dependency:
it is plain CUDA runtime code behind a C ABI (see ``include/dyllm_b200.h``).  The binding links to neither: Python hands it the
library's entry points.
"""

from __future__ import annotations

import hashlib
import os
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

PKG_DIR = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(PKG_DIR, "csrc")
INCLUDE = os.path.join(os.path.dirname(PKG_DIR), "include")
LIB_PATH = os.path.join(PKG_DIR, "libdyllm_b200.so")
BINDING_PATH = os.path.join(PKG_DIR, "_native.so")
OBJ_DIR = os.path.join(PKG_DIR, "build")

NVCC_FLAGS = [
    "-gencode",
    "arch=compute_100a,code=sm_100a",
    "-O3",
    "-std=c++17",
    "-lineinfo",
    "--use_fast_math",
    "-Xcompiler",
    "-fPIC",
]


def _nvcc() -> str:
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(nvcc):
        raise RuntimeError("nvcc not found; dyllm_b200 cannot be built")
    return nvcc


def sources() -> list[str]:
    return sorted(os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith(".cu"))


def _digest(path: str) -> str:
    h = hashlib.sha256()
    for dep in [path] + sorted(
        os.path.join(d, f) for d in (CSRC, INCLUDE) for f in os.listdir(d) if f.endswith((".cuh", ".h"))
    ):
        with open(dep, "rb") as fh:
            h.update(fh.read())
    h.update(" ".join(NVCC_FLAGS).encode())
    return h.hexdigest()


def _compile_one(src: str, verbose: bool) -> tuple[str, bool]:
    obj = os.path.join(OBJ_DIR, os.path.basename(src)[:-3] + ".o")
    stamp = obj + ".sha"
    digest = _digest(src)
    if os.path.exists(obj) and os.path.exists(stamp) and open(stamp).read() == digest:
        return obj, False
    cmd = [_nvcc(), *NVCC_FLAGS, "-I", INCLUDE, "-c", src, "-o", obj]
    if verbose:
        cmd.insert(1, "-Xptxas")
        cmd.insert(2, "-v")
    res = subprocess.run(cmd, capture_output=True, text=True)
    if verbose or res.returncode != 0:
        sys.stderr.write(res.stdout + res.stderr)
    if res.returncode != 0:
        raise RuntimeError(f"nvcc failed for {src}")
    with open(stamp, "w") as fh:
        fh.write(digest)
    return obj, True


def _build_binding(verbose: bool) -> None:
    import sysconfig

    import torch

    src, stamp = os.path.join(CSRC, "bind.cpp"), os.path.join(OBJ_DIR, "bind.sha")
    h = hashlib.sha256(f"{torch.__version__} {sys.version}".encode())
    for dep in (src, os.path.join(INCLUDE, "dyllm_b200.h")):
        with open(dep, "rb") as fh:
            h.update(fh.read())
    if os.path.exists(BINDING_PATH) and os.path.exists(stamp) and open(stamp).read() == h.hexdigest():
        return
    tdir = os.path.dirname(torch.__file__)
    cuda = os.path.dirname(os.path.dirname(os.path.realpath(_nvcc())))
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           "-I", INCLUDE, "-isystem", f"{tdir}/include", "-isystem", f"{tdir}/include/torch/csrc/api/include", "-isystem", f"{cuda}/include",
           "-isystem", sysconfig.get_path("include"), src, "-o", BINDING_PATH, "-L", f"{tdir}/lib", "-lc10", "-lc10_cuda", "-ltorch_cpu",
           "-ltorch_python"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if verbose or res.returncode != 0:
        sys.stderr.write(res.stdout + res.stderr)
    if res.returncode != 0:
        raise RuntimeError(f"the C++ compiler failed for {src}")
    with open(stamp, "w") as fh:
        fh.write(h.hexdigest())


def build(force: bool = False, verbose: bool = False) -> str:
    os.makedirs(OBJ_DIR, exist_ok=True)
    if force:
        for f in os.listdir(OBJ_DIR):
            os.remove(os.path.join(OBJ_DIR, f))
    srcs = sources()
    with ThreadPoolExecutor(max_workers=min(9, len(srcs) + 1)) as pool:
        binding = pool.submit(_build_binding, verbose)
        results = list(pool.map(lambda s: _compile_one(s, verbose), srcs))
        binding.result()
    objs = [o for o, _ in results]
    if any(changed for _, changed in results) or not os.path.exists(LIB_PATH):
        cmd = [_nvcc(), "-shared", "-o", LIB_PATH, *objs, "-gencode", "arch=compute_100a,code=sm_100a",
               "-Xcompiler", "-fPIC"]
        res = subprocess.run(cmd, capture_output=True, text=True)
        if res.returncode != 0:
            sys.stderr.write(res.stdout + res.stderr)
            raise RuntimeError("linking libdyllm_b200.so failed")
    return LIB_PATH


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="--verbose" in sys.argv))
