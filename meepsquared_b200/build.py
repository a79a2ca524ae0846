"""Builds libmeep2b.so in the package directory with nvcc for sm_100a (B200) only, and _native.so, the autograd nodes that
call it, with the host compiler against the installed torch.

    python -m meepsquared_b200.build [--verbose]

The library is one translation unit (csrc/libmeep2b.cu) with the CUDA runtime linked statically, so it loads
without the driver library present; it resolves cuTensorMapEncodeTiled through the runtime at first use.
"""

import os
import shutil
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
LIB = os.path.join(HERE, "libmeep2b.so")
SOURCES = ["libmeep2b.cu", "capi.cu", "route.cu", "grouped_gemm.cu", "grouped_gemm_q.cuh", "grouped_gemm_qpair.cuh",
           "reduce.cu", "quant.cu", "merge.cu", "fp8_products.cu", "swiglu.cu", "vocab_loss.cu",
           "balance.cu", "head_norm.cu",
           "common.cuh", "host.hpp"]


NATIVE = os.path.join(HERE, "_native.so")
NATIVE_SOURCE = os.path.join(HERE, "csrc", "native.cpp")


def nvcc() -> str:
    for c in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if c and os.path.exists(c):
            return c
    raise RuntimeError("nvcc not found: the CUDA toolkit is needed to build libmeep2b")


def stale() -> bool:
    if not os.path.exists(LIB):
        return True
    t = os.path.getmtime(LIB)
    deps = [os.path.join(HERE, "csrc", s) for s in SOURCES] + [os.path.join(HERE, "..", "include", "meep2b.h")]
    return any(os.path.getmtime(d) > t for d in deps if os.path.exists(d))


def build(verbose: bool = False, force: bool = False) -> str:
    if force or stale():
        build_library(verbose)
    if force or native_stale():
        build_native(verbose)
    return LIB


def native_tag() -> str:
    """What the autograd nodes' layout depends on (torch, its C++ ABI, the interpreter's): _native.so holds it."""
    import torch

    return f"built for torch {torch.__version__}, ABI {int(torch._C._GLIBCXX_USE_CXX11_ABI)}, " \
           f"{sysconfig.get_config_var('EXT_SUFFIX')}"


def native_stale() -> bool:
    if not os.path.exists(NATIVE):
        return True
    with open(NATIVE, "rb") as f:
        if native_tag().encode() not in f.read():
            return True
    t = os.path.getmtime(NATIVE)
    return any(os.path.getmtime(d) > t for d in (NATIVE_SOURCE, os.path.join(HERE, "..", "include", "meep2b.h")))


def build_native(verbose: bool = False) -> str:
    import torch

    cxx = os.environ.get("CXX") or shutil.which("g++") or "c++"
    root = os.path.dirname(torch.__file__)
    cuda = os.path.dirname(os.path.dirname(os.path.realpath(nvcc())))
    includes = [os.path.join(root, "include"), os.path.join(root, "include", "torch", "csrc", "api", "include"),
                sysconfig.get_paths()["include"], os.path.join(cuda, "include")]
    cmd = [cxx, "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden", "-DTORCH_EXTENSION_NAME=_native",
           f'-DMEEP2B_NATIVE_TAG="{native_tag()}"',
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", *[f"-I{d}" for d in includes], NATIVE_SOURCE,
           "-o", NATIVE + ".tmp", f"-L{HERE}", "-l:" + os.path.basename(LIB), "-L" + os.path.join(root, "lib"), "-lc10",
           "-lc10_cuda", "-ltorch", "-ltorch_cpu", "-ltorch_python", "-Wl,-rpath,$ORIGIN"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError("the host compiler failed:\n" + r.stdout + r.stderr)
    if verbose:
        sys.stderr.write(r.stdout + r.stderr)
    os.replace(NATIVE + ".tmp", NATIVE)
    return NATIVE


def build_library(verbose: bool = False) -> str:
    cmd = [nvcc(), "-gencode", "arch=compute_100a,code=sm_100a", "-O3", "-lineinfo", "-std=c++17",
           "--expt-relaxed-constexpr", "-Xcompiler", "-fPIC", "-shared", "-cudart", "static",
           "-o", LIB + ".tmp", os.path.join(HERE, "csrc", "libmeep2b.cu")]
    if verbose:
        cmd.insert(1, "-Xptxas=-v")
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError("nvcc failed:\n" + r.stdout + r.stderr)
    if verbose:
        sys.stderr.write(r.stdout + r.stderr)
    os.replace(LIB + ".tmp", LIB)
    return LIB


if __name__ == "__main__":
    print(build(verbose="--verbose" in sys.argv, force=True))
