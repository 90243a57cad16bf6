"""Build the in-tree CUDA libraries for sm_100a (nvcc cross-compiles; no GPU
needed).  Outputs land next to the Python package that loads them, so they
travel with the repository snapshot.

    python gpu-forge_b200/build.py            # build what is out of date
    python gpu-forge_b200/build.py --force    # rebuild everything
"""
from __future__ import annotations

import concurrent.futures
import os
import subprocess
import sys

PKG = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG)
CSRC = os.path.join(PKG, "csrc")
INCLUDE = os.path.join(ROOT, "include")
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC", "-I" + INCLUDE, "-I" + CSRC]

# target -> its sources, each with the headers of csrc/ it includes; the
# public headers go for all of them
TARGETS = {
    os.path.join(PKG, "forge_sort", "libforgesort.so"): {
        "srcs": {
            "fs_sort.cu": ["fs_internal.h", "fs_device.cuh", "fs_kernels.cuh", "fs_histfill.cuh", "fs_resident.cuh",
                           "fs_hoststage.h"],
            "fs_multi.cu": ["fs_device.cuh"],
            "fs_datagen.cu": ["fs_device.cuh"],
            "fs_rows.cu": ["fs_internal.h", "fs_device.cuh", "fs_rows.cuh"],
            "fs_slots.cu": ["fs_internal.h", "fs_device.cuh"],
        },
        "hdrs": ["forgesort.h", "forgesort_bench.h"],
        "libs": [],
    },
}
OBJ = os.path.join(PKG, "build")  # one object per source: a change recompiles what includes it


def _stale(target: str, inputs) -> bool:
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(p) > t for p in inputs)


def _run(cmd, verbose: bool) -> None:
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.run(cmd, check=True)


def build(force: bool = False, verbose: bool = False) -> None:
    for target, spec in TARGETS.items():
        hdrs = [os.path.join(INCLUDE, h) for h in spec["hdrs"]]
        inputs = {src: [os.path.join(CSRC, f) for f in (src, *deps)] + hdrs for src, deps in spec["srcs"].items()}
        if not force and not _stale(target, [p for ps in inputs.values() for p in ps]):
            continue
        os.makedirs(OBJ, exist_ok=True)
        objs = {src: os.path.join(OBJ, os.path.splitext(src)[0] + ".o") for src in inputs}
        todo = [[NVCC, *ARCH, *FLAGS, "-c", os.path.join(CSRC, src), "-o", obj] for src, obj in objs.items()
                if force or _stale(obj, inputs[src])]
        with concurrent.futures.ThreadPoolExecutor(max_workers=max(1, os.cpu_count() or 1)) as pool:
            list(pool.map(lambda cmd: _run(cmd, verbose), todo))
        _run([NVCC, *ARCH, "-shared", "-Xcompiler", "-fPIC", *objs.values(), "-o", target, *spec["libs"]], verbose)


if __name__ == "__main__":
    build(force="--force" in sys.argv, verbose=True)
