"""Build libdeltacore.so in-tree for sm_100a with nvcc.

    python burn-deltanet_b200/build.py          # incremental (skips when up to date)
    python burn-deltanet_b200/build.py --force

The library is the C ABI of include/deltacore.h and include/deltacore_layers.h.  Its translation units
(csrc/*.cu) are compiled side by side into _build/ and linked in the package directory, so that it travels
with the source tree; nothing is installed.
"""
from __future__ import annotations

import glob
import os
import re
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libdeltacore.so")
OBJ = os.path.join(HERE, "_build")
ARCH = "-gencode=arch=compute_100a,code=sm_100a"


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found: the delta-rule core needs the CUDA toolkit to build")


def units() -> list[str]:
    """The translation units of the library."""
    return sorted(glob.glob(os.path.join(CSRC, "*.cu")))


def sources() -> list[str]:
    return sorted(units() + glob.glob(os.path.join(CSRC, "*.cuh")) + glob.glob(os.path.join(CSRC, "*.hpp"))
                  + glob.glob(os.path.join(ROOT, "include", "*.h")))


def included(path: str, seen: set[str] | None = None) -> set[str]:
    """`path` and the files of this tree that it includes, directly or not."""
    seen = set() if seen is None else seen
    path = os.path.normpath(path)
    if path not in seen and os.path.exists(path):
        seen.add(path)
        with open(path) as f:
            for name in re.findall(r'#include "([^"]+)"', f.read()):
                included(os.path.join(os.path.dirname(path), name), seen)
    return seen


def newer(target: str, deps) -> bool:
    return os.path.exists(target) and all(os.path.getmtime(d) <= os.path.getmtime(target) for d in deps)


def up_to_date() -> bool:
    return newer(LIB, sources())


def compile_unit(src: str, force: bool, verbose: bool) -> str:
    obj = os.path.join(OBJ, os.path.splitext(os.path.basename(src))[0] + ".o")
    if force or not newer(obj, included(src)):
        cmd = [
            nvcc(), ARCH, "-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC",
            "-Xcompiler", "-fvisibility=hidden", "-Xptxas", "-v" if verbose else "-O3",
            "--expt-relaxed-constexpr", "-I", os.path.join(ROOT, "include"), "-c", src, "-o", obj + ".tmp",
        ]
        subprocess.run(cmd, check=True)
        os.replace(obj + ".tmp", obj)
    return obj


def build(force: bool = False, verbose: bool = False) -> str:
    if not force and up_to_date():
        return LIB
    os.makedirs(OBJ, exist_ok=True)
    with ThreadPoolExecutor(max_workers=os.cpu_count() or 1) as pool:
        objs = list(pool.map(lambda src: compile_unit(src, force, verbose), units()))
    subprocess.run([nvcc(), ARCH, "--shared", "-Xcompiler", "-fPIC", *objs, "-o", LIB + ".tmp", "-lcuda"], check=True)
    os.replace(LIB + ".tmp", LIB)
    return LIB


if __name__ == "__main__":
    build(force="--force" in sys.argv, verbose="-v" in sys.argv)
    print(LIB)
