"""Build libsdcguard_hip.so (gfx950) in-tree from the .hip sources next to this file.

    python -m sdcguard_amd.csrc.build          # or sdcguard_amd.csrc.build.build()

Every source is compiled with hipcc for gfx950 only, packed-fp32 instructions disabled, then linked into
sdcguard_amd/libsdcguard_hip.so, which sdcguard_amd._lib loads with ctypes.  bind.cpp, host code against torch's headers,
becomes the extension module sdcguard_amd/_bind.so.
"""
from __future__ import annotations

import concurrent.futures as cf
import glob
import os
import shutil
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
PKG = os.path.dirname(HERE)
LIB = os.path.join(PKG, "libsdcguard_hip.so")
BIND = os.path.join(PKG, "_bind.so")
OBJDIR = os.path.join(PKG, "_build")
ARCH = os.environ.get("SDCGUARD_HIP_ARCH", "gfx950")

FLAGS = ["-O3", "-std=c++17", "-fPIC", f"--offload-arch={ARCH}", "-ffp-contract=fast",
         # packed fp32 VALU forms are kept out of every kernel
         "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
         "-Wno-unused-command-line-argument"]


def _hipcc() -> str:
    for cand in (os.environ.get("HIPCC"), shutil.which("hipcc"), "/opt/rocm/bin/hipcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("hipcc not found: the sdcguard HIP library cannot be built")


def sources() -> list:
    return sorted(glob.glob(os.path.join(HERE, "*.hip")))


def _compile(src: str) -> str:
    obj = os.path.join(OBJDIR, os.path.basename(src)[:-4] + ".o")
    cmd = [_hipcc(), *FLAGS, "-I", HERE, "-c", src, "-o", obj]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"hipcc failed on {os.path.basename(src)}:\n{r.stderr[-6000:]}")
    return obj


def _bind() -> None:
    import torch
    root = os.path.dirname(os.path.abspath(torch.__file__))
    rocm = os.path.dirname(os.path.dirname(os.path.realpath(_hipcc())))
    tmp = BIND + ".tmp"
    # -D: what HIP's host headers ask of a compiler that is not hipcc
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-D__HIP_PLATFORM_AMD__",
           "-I", os.path.join(root, "include"), "-I", os.path.join(root, "include", "torch", "csrc", "api", "include"),
           "-I", sysconfig.get_paths()["include"], "-I", os.path.join(rocm, "include"), os.path.join(HERE, "bind.cpp"),
           "-o", tmp, "-L", os.path.join(root, "lib"), "-lc10", "-lc10_hip", "-ltorch_cpu", "-ltorch_python"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"g++ failed on bind.cpp:\n{r.stderr[-6000:]}")
    os.replace(tmp, BIND)


def build(verbose: bool = False) -> str:
    os.makedirs(OBJDIR, exist_ok=True)
    srcs = sources()
    with cf.ThreadPoolExecutor(max_workers=min(8, len(srcs) + 1)) as ex:
        bind = ex.submit(_bind)
        objs = list(ex.map(_compile, srcs))
        bind.result()
    tmp = LIB + ".tmp"
    cmd = [_hipcc(), f"--offload-arch={ARCH}", "-shared", "-fPIC", "-o", tmp, *objs]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{r.stderr[-6000:]}")
    os.replace(tmp, LIB)
    if verbose:
        print(f"built {LIB} from {len(srcs)} sources")
    return LIB


if __name__ == "__main__":
    build(verbose=True)
    sys.exit(0)
