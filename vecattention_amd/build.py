"""Build libvecattn.so (the HIP kernels + C ABI) in-tree for gfx950, and the
host module _host.so (csrc/host_calls.cpp) on top of it.

Usage: python -m vecattention_amd.build [--jobs N]
The library lands next to this file, so it travels with the source tree.
"""
import argparse
import os
import shutil
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor

import torch

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libvecattn.so")
HOST = os.path.join(HERE, "_host.so")
SOURCES = ["pool.hip", "select_exact.hip", "select_mfma.hip", "select_tile.hip", "select_max.hip",
           "select_wave.hip", "key_norm.hip",
           "attn_simple.hip", "attn_mfma.hip", "attn_dense.hip", "attn_f32.hip", "decode.hip",
           "csr.hip", "convert.hip", "paged_plan.hip", "rope.hip", "paged_attn.hip",
           "paged_prefix.hip", "paged_share.hip", "paged_copy.hip", "paged_api.hip",
           "api.hip", "noalloc.hip"]
ARCH = os.environ.get("VA_OFFLOAD_ARCH", "gfx950")

# -packed-fp32-ops: no v_pk_{add,mul,fma}_f32 are generated (they have given
# silently wrong results on the target machines).  -ffp-contract=off keeps the
# canonical (un-fused) rounding of the selection arithmetic.
FLAGS = [
    f"--offload-arch={ARCH}", "-O3", "-std=c++17", "-fPIC", "-ffp-contract=off",
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-Wall", "-Wno-unused-result",
]


def hipcc():
    exe = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(exe):
        raise RuntimeError("hipcc not found; the HIP toolchain is required to build libvecattn.so")
    return exe


def _compile(src, build_dir):
    obj = os.path.join(build_dir, os.path.splitext(src)[0] + ".o")
    cmd = [hipcc(), *FLAGS, "-c", os.path.join(CSRC, src), "-o", obj]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"hipcc failed for {src}:\n{r.stderr}")
    return obj


def _run(what, cmd):
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"{what} failed:\n{r.stderr}")


def _compile_host(build_dir):
    """csrc/host_calls.cpp, plain C++ against torch's and Python's headers."""
    from torch.utils.cpp_extension import include_paths
    obj = os.path.join(build_dir, "host_calls.o")
    dirs = [*include_paths(), sysconfig.get_paths()["include"]]
    _run("the compiler for host_calls.cpp",
         [shutil.which("g++") or hipcc(), "-O2", "-std=c++17", "-fPIC", "-Wall",
          f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
          *(a for d in dirs for a in ("-isystem", d)), "-c",
          os.path.join(CSRC, "host_calls.cpp"), "-o", obj])
    return obj


def _link_host(obj):
    libs = os.path.join(os.path.dirname(torch.__file__), "lib")
    _run("link of _host.so",
         [shutil.which("g++") or hipcc(), "-shared", "-o", HOST + ".tmp", obj, f"-L{HERE}",
          "-l:libvecattn.so", "-Wl,-rpath,$ORIGIN", f"-L{libs}", "-ltorch_python", "-ltorch_cpu",
          "-lc10"])
    os.replace(HOST + ".tmp", HOST)


def build(jobs=None, verbose=False):
    build_dir = os.path.join(HERE, "_build")
    os.makedirs(build_dir, exist_ok=True)
    jobs = jobs or min(len(SOURCES), os.cpu_count() or 1)
    with ThreadPoolExecutor(max_workers=jobs) as ex:
        host = ex.submit(_compile_host, build_dir)
        objs = list(ex.map(lambda s: _compile(s, build_dir), SOURCES))
    tmp = LIB + ".tmp"
    cmd = [hipcc(), f"--offload-arch={ARCH}", "-shared", "-fPIC", "-o", tmp, *objs]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{r.stderr}")
    os.replace(tmp, LIB)
    _link_host(host.result())
    if verbose:
        print(f"built {LIB}")
    return LIB


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--jobs", type=int, default=None)
    a = ap.parse_args()
    build(a.jobs, verbose=True)
    sys.exit(0)
