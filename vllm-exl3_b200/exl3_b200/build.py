"""Build the sm_100a shared library ``libexl3_b200.so`` in-tree with nvcc, and
``_serving_py.*.so``, the short way from Python into its serving entries, with g++.

The library exports the C ABI declared in ``include/exl3_b200.h``; it is
loaded with ctypes by :mod:`exl3_b200._native`.  The CUDA runtime is linked
statically so the library does not depend on which libcudart the host
process loaded first.
"""

from __future__ import annotations

import os
import shutil
import subprocess

PKG_DIR = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG_DIR)
CSRC = os.path.join(ROOT, "csrc")
LIB_PATH = os.path.join(PKG_DIR, "libexl3_b200.so")
BINDING_SRC = os.path.join(CSRC, "serving_py.cpp")

SOURCES = ["capi.cu", "moe.cu", "reconstruct.cu", "noalloc.cu", "tc_gemm.cu", "ep.cu", "ngram.cu",
           "kv_cache.cu", "kv_attend.cu", "kv_prompt.cu", "logprobs.cu"]
HEADERS = ["exl3_common.cuh", "exl3_internal.h", "tc_common.cuh", "tc_gemm.h", "kv_common.cuh", "kv_attend.cuh"]

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-lineinfo", "-O3", "-std=c++17",
    "-Xcompiler", "-fPIC", "-shared",
    "-cudart", "static",
]


def _nvcc() -> str:
    cand = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(cand):
        raise RuntimeError("nvcc not found: the EXL3 CUDA library cannot be built")
    return cand


def _inputs() -> list[str]:
    hdr = os.path.join(os.path.dirname(ROOT), "include", "exl3_b200.h")
    return [os.path.join(CSRC, s) for s in SOURCES + HEADERS] + [hdr]


def binding_path() -> str:
    """The serving binding's file, named by what it is compiled against: this interpreter's ABI and torch's version."""
    import sysconfig

    import torch
    return os.path.join(PKG_DIR, f"_serving_py.{sysconfig.get_config_var('SOABI')}.torch-{torch.__version__}.so")


def build_binding(force: bool = False, verbose: bool = False) -> str:
    """Compile the serving binding against this interpreter and its torch."""
    path = binding_path()
    hdr = os.path.join(os.path.dirname(ROOT), "include", "exl3_b200.h")
    if not force and os.path.exists(path) and \
            os.path.getmtime(path) >= max(os.path.getmtime(p) for p in (BINDING_SRC, hdr)):
        return path
    import sysconfig

    import torch
    home = os.path.dirname(torch.__file__)
    include = [sysconfig.get_paths()["include"], os.path.join(home, "include"),
               os.path.join(home, "include", "torch", "csrc", "api", "include"),
               os.path.join(os.path.dirname(os.path.dirname(os.path.realpath(_nvcc()))), "include")]
    tmp = f"{path}.{os.getpid()}.tmp"  # processes may build at once
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", *(f"-I{i}" for i in include),
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", BINDING_SRC, "-o", tmp,
           f"-L{os.path.join(home, 'lib')}", "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_python"]
    if verbose:
        print(" ".join(cmd), flush=True)
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"g++ failed ({res.returncode}):\n{res.stderr[-4000:]}")
    os.replace(tmp, path)
    return path


def up_to_date() -> bool:
    if not os.path.exists(LIB_PATH):
        return False
    t = os.path.getmtime(LIB_PATH)
    return all(os.path.getmtime(p) <= t for p in _inputs() if os.path.exists(p))


def build(force: bool = False, verbose: bool = False) -> str:
    """Compile the library if any source is newer; returns its path."""
    if not force and up_to_date():
        return LIB_PATH
    tmp = f"{LIB_PATH}.{os.getpid()}.tmp"
    cmd = [_nvcc(), *NVCC_FLAGS, "-o", tmp, *[os.path.join(CSRC, s) for s in SOURCES]]
    if verbose:
        print(" ".join(cmd), flush=True)
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"nvcc failed ({res.returncode}):\n{res.stderr[-4000:]}")
    os.replace(tmp, LIB_PATH)
    return LIB_PATH


if __name__ == "__main__":
    print(build(force=True, verbose=True))
    print(build_binding(force=True, verbose=True))
