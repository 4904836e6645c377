"""Build libkvx.so in-tree for sm_100a with nvcc.

``python -m aegaeon_b200.build`` (or ``__graft_entry__.build()``).  The
library links the CUDA runtime statically so that it does not depend on which
libcudart another extension in the process loaded first.
"""

from __future__ import annotations

import os
import shutil
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
SOURCES = [
    os.path.join(HERE, "csrc", "kvx_plan.cpp"),
    os.path.join(HERE, "csrc", "kvx_runtime.cu"),
    os.path.join(HERE, "csrc", "kvx_noalloc.cu"),
    os.path.join(HERE, "csrc", "kvx_safetensors.cpp"),
    os.path.join(HERE, "csrc", "kvx_events.cu"),
    os.path.join(HERE, "csrc", "kvx_q4.cu"),
]
HEADERS = [
    os.path.join(HERE, "csrc", "kvx_plan.h"),
    os.path.join(HERE, "csrc", "kvx_worklist.h"),
    os.path.join(HERE, "csrc", "kvx_kernels.cuh"),
    os.path.join(HERE, "csrc", "kvx_q4_rows.cuh"),
    os.path.join(HERE, "csrc", "kvx_q4_attention.cuh"),
    os.path.join(HERE, "csrc", "kvx_q4_extend.cuh"),
    os.path.join(ROOT, "include", "kvx.h"),
]
OUT = os.path.join(HERE, "libkvx.so")
SHIM_SOURCE = os.path.join(HERE, "csrc", "kvx_pycall.c")
SHIM_OUT = os.path.join(HERE, "_kvxcall" + sysconfig.get_config_var("EXT_SUFFIX"))
Q4_SOURCE = os.path.join(HERE, "csrc", "kvx_q4_torch.cpp")
Q4_OUT = os.path.join(HERE, "_kvxq4" + sysconfig.get_config_var("EXT_SUFFIX"))
ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found")


def up_to_date() -> bool:
    if not os.path.exists(OUT):
        return False
    t = os.path.getmtime(OUT)
    return all(os.path.getmtime(p) <= t for p in SOURCES + HEADERS)


def build_shim(force: bool = False) -> str:
    """The Python call shim (plain C against the CPython headers; it reaches
    libkvx.so through function pointers handed over at import)."""
    deps = [SHIM_SOURCE, os.path.join(ROOT, "include", "kvx.h")]
    if (not force and os.path.exists(SHIM_OUT)
            and all(os.path.getmtime(p) <= os.path.getmtime(SHIM_OUT) for p in deps)):
        return SHIM_OUT
    cc = os.environ.get("CC") or shutil.which("gcc") or "cc"
    cmd = [cc, "-O2", "-Wall", "-shared", "-fPIC", "-I" + sysconfig.get_paths()["include"],
           SHIM_SOURCE, "-o", SHIM_OUT + ".tmp"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"{cc} failed ({res.returncode}):\n{res.stderr}\n{res.stdout}")
    os.replace(SHIM_OUT + ".tmp", SHIM_OUT)
    return SHIM_OUT


def build_q4_module(force: bool = False) -> str:
    """The tensor entry points of the 4-bit cache (C++ against torch's headers;
    it reaches libkvx.so through function pointers handed over at import)."""
    deps = [Q4_SOURCE, os.path.join(ROOT, "include", "kvx.h")]
    if (not force and os.path.exists(Q4_OUT)
            and all(os.path.getmtime(p) <= os.path.getmtime(Q4_OUT) for p in deps)):
        return Q4_OUT
    import torch

    cxx = os.environ.get("CXX") or shutil.which("g++") or "c++"
    cuda = os.path.join(os.path.dirname(os.path.dirname(os.path.realpath(nvcc()))), "include")
    home = os.path.dirname(torch.__file__)
    includes = [sysconfig.get_paths()["include"], cuda, os.path.join(home, "include"),
                os.path.join(home, "include", "torch", "csrc", "api", "include")]
    lib = os.path.join(home, "lib")
    cmd = [cxx, "-O2", "-std=c++17", "-Wall", "-shared", "-fPIC",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}",
           *(f"-isystem{p}" for p in includes), Q4_SOURCE, f"-L{lib}", "-ltorch_python",
           "-ltorch_cpu", "-lc10_cuda", "-lc10", "-o", Q4_OUT + ".tmp"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"{cxx} failed ({res.returncode}):\n{res.stderr}\n{res.stdout}")
    os.replace(Q4_OUT + ".tmp", Q4_OUT)
    return Q4_OUT


def build(force: bool = False, verbose: bool = False) -> str:
    build_shim(force)
    build_q4_module(force)
    if not force and up_to_date():
        return OUT
    cmd = [
        nvcc(), "-O3", "-std=c++17", *ARCH_FLAGS, "-lineinfo",
        "-Xcompiler", "-fPIC,-Wall", "-shared", "-cudart", "static",
        *SOURCES, "-o", OUT + ".tmp",
    ]
    if verbose:
        cmd.insert(1, "-Xptxas=-v")
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"nvcc failed ({res.returncode}):\n{res.stderr}\n{res.stdout}")
    if verbose:
        sys.stderr.write(res.stderr)
    os.replace(OUT + ".tmp", OUT)
    return OUT


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
