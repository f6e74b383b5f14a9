"""Build libnsattn.so in-tree for sm_100a with nvcc (no JIT cache, no setuptools), and _native, the Python binding
of its decode operators, with g++ against torch's headers.

    python -m nanosaur2_web_b200.build [--verbose]

Both shared libraries land next to this file so they travel with the source tree; the C ABI is
declared in include/nsattn.h.
"""

from __future__ import annotations

import argparse
import os
import shutil
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
INCLUDE = os.path.join(ROOT, "include")
LIB = os.path.join(HERE, "libnsattn.so")
BINDING = os.path.join(HERE, "_native" + sysconfig.get_config_var("EXT_SUFFIX"))
SOURCES = ["api.cu", "attention.cu", "attention_persist.cu", "attention_d512.cu", "prologue.cu", "no_alloc.cu", "proj.cu", "linear.cu", "rmsnorm.cu", "glu.cu", "rotate.cu", "lora.cu",
           "linear4.cu", "kv4.cu"]
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]


def nvcc_path() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found: the CUDA 12.9 toolkit is required to build libnsattn.so")


def build_binding(force: bool = False) -> str:
    """The C++ binding over torch tensors; links libnsattn.so next to it."""
    src = os.path.join(CSRC, "binding.cpp")
    header = os.path.join(INCLUDE, "nsattn.h")
    if not force and os.path.exists(BINDING) and all(os.path.getmtime(BINDING) >= os.path.getmtime(d) for d in (src, header)):
        return BINDING
    import torch
    from torch.utils.cpp_extension import include_paths, library_paths
    inc = [INCLUDE, sysconfig.get_paths()["include"], *include_paths(device_type="cuda")]
    libs = library_paths(device_type="cuda")
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-shared", "-fPIC", "-fvisibility=hidden",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           *[a for i in inc for a in ("-isystem", i)], src, "-o", BINDING + ".tmp",
           *[f"-L{p}" for p in libs], f"-L{HERE}", "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch", "-ltorch_python",
           "-l:libnsattn.so", "-Wl,-rpath,$ORIGIN"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        sys.stderr.write(res.stdout + res.stderr)
        raise RuntimeError("g++ failed building the Python binding")
    os.replace(BINDING + ".tmp", BINDING)
    return BINDING


def build(verbose: bool = False, force: bool = False) -> str:
    lib = build_library(verbose, force)
    build_binding(force)
    return lib


def build_library(verbose: bool = False, force: bool = False) -> str:
    srcs = [os.path.join(CSRC, s) for s in SOURCES]
    deps = srcs + [os.path.join(CSRC, h) for h in os.listdir(CSRC) if h.endswith((".h", ".cuh"))]
    deps.append(os.path.join(INCLUDE, "nsattn.h"))
    if not force and os.path.exists(LIB) and all(os.path.getmtime(LIB) >= os.path.getmtime(d) for d in deps):
        return LIB
    cmd = [nvcc_path(), *ARCH, "-O3", "-lineinfo", "-std=c++17", "-shared", "-Xcompiler", "-fPIC,-O3",
           "-I", INCLUDE, "-I", CSRC, "-o", LIB + ".tmp", *srcs]
    if verbose:
        cmd += ["-Xptxas", "-v"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        sys.stderr.write(res.stdout + res.stderr)
        raise RuntimeError("nvcc failed building libnsattn.so")
    if verbose:
        sys.stderr.write(res.stderr)
    os.replace(LIB + ".tmp", LIB)
    return LIB


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--verbose", action="store_true")
    ap.add_argument("--force", action="store_true")
    a = ap.parse_args()
    print(build(verbose=a.verbose, force=a.force))
