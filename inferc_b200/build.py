"""Builds libinferc_b200.so in-tree with nvcc for sm_100a (B200 only), and the
torch binding of the paged-cache operators (csrc/torch_paged.cpp) against it.

    python -m inferc_b200.build [--force]

Objects go to inferc_b200/_build/, the shared library to
inferc_b200/libinferc_b200.so and the binding to inferc_b200/_paged.so; all are
git-ignored build products. Without torch the binding is left out; the library
needs nvcc alone.
"""
from __future__ import annotations

import argparse
import concurrent.futures as cf
import glob
import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
BUILD = os.path.join(HERE, "_build")
LIB = os.path.join(HERE, "libinferc_b200.so")
BINDING = os.path.join(HERE, "_paged.so")
INCLUDE = os.path.join(os.path.dirname(HERE), "include")
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC", "-Xcompiler", "-Wall",
         "--expt-relaxed-constexpr", f"-I{INCLUDE}"]


def _deps() -> list[str]:
    return (glob.glob(os.path.join(CSRC, "*.cuh")) + glob.glob(os.path.join(CSRC, "*.h")) +
            glob.glob(os.path.join(INCLUDE, "*.h")))


def _stale(target: str, sources: list[str]) -> bool:
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(s) > t for s in sources)


def _compile(src: str, force: bool, verbose_ptxas: bool) -> str:
    obj = os.path.join(BUILD, os.path.basename(src) + ".o")
    if force or _stale(obj, [src] + _deps()):
        cmd = [NVCC, *ARCH, *FLAGS, "-c", src, "-o", obj]
        if verbose_ptxas:
            cmd.insert(1, "-Xptxas=-v")
        subprocess.run(cmd, check=True)
    return obj


def _build_binding(force: bool) -> None:
    """The torch binding; without torch the library stands alone, as its C ABI does."""
    src = os.path.join(CSRC, "torch_paged.cpp")
    if not (force or _stale(BINDING, [src, LIB] + _deps())):
        return
    import sysconfig

    try:
        import torch
    except ImportError:
        print(f"torch is not installed: {os.path.basename(BINDING)} (the paged-cache operators of "
              "inferc_b200.ops) is not built", file=sys.stderr)
        return
    root = os.path.dirname(torch.__file__)
    inc = [os.path.join(root, "include"), os.path.join(root, "include", "torch", "csrc", "api",
                                                       "include"),
           sysconfig.get_paths()["include"],
           os.path.join(os.path.dirname(os.path.dirname(NVCC)), "include")]
    subprocess.run(
        ["g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-w",
         f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
         *[f"-I{i}" for i in inc], src, "-o", BINDING, LIB, f"-L{os.path.join(root, 'lib')}",
         "-ltorch_python", "-ltorch_cuda", "-ltorch_cpu", "-ltorch", "-lc10_cuda", "-lc10",
         "-Wl,-rpath,$ORIGIN", f"-Wl,-rpath,{os.path.join(root, 'lib')}"], check=True)


def build(force: bool = False, verbose_ptxas: bool = False) -> str:
    os.makedirs(BUILD, exist_ok=True)
    sources = sorted(glob.glob(os.path.join(CSRC, "*.cu")) + glob.glob(os.path.join(CSRC, "*.cc")))
    with cf.ThreadPoolExecutor(max_workers=min(8, os.cpu_count() or 1)) as ex:
        objs = list(ex.map(lambda s: _compile(s, force, verbose_ptxas), sources))
    if force or _stale(LIB, objs):
        subprocess.run([NVCC, *ARCH, "-shared", "-o", LIB, "-Xlinker",
                        "-soname=libinferc_b200.so", *objs, "-lcudart"], check=True)
    _build_binding(force)
    return LIB


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--ptxas-v", action="store_true")
    a = ap.parse_args()
    print(build(a.force, a.ptxas_v), file=sys.stderr)
