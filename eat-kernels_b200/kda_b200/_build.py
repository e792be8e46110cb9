"""Builds libkda_b200.so in-tree with nvcc for sm_100a (explicit -gencode; no JIT cache, no torch dependency)."""
from __future__ import annotations

import os
import shutil
import subprocess
import tempfile
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PKG = Path(__file__).resolve().parent
CSRC = PKG.parent / "csrc"
LIB = PKG / "libkda_b200.so"
SOURCES = ["kda_chunk_umma.cu", "kda_chunk_fwd.cu", "kda_plan.cu", "kda_cp.cu", "kda_conv.cu", "kda_sscan.cu", "kda_step.cu",
           "kda_pool.cu", "kda_capi.cu"]
NVCC_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17", "-Xcompiler", "-fPIC"]


def nvcc_path() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("nvcc not found: libkda_b200.so cannot be built")


def stale() -> bool:
    if not LIB.exists():
        return True
    t = LIB.stat().st_mtime
    deps = list(CSRC.glob("*.cu")) + list(CSRC.glob("*.cuh")) + [PKG.parent.parent / "include" / "kda_b200.h"]
    return any(d.stat().st_mtime > t for d in deps)


def build_library(force: bool = False, verbose: bool = False) -> Path:
    if not force and not stale():
        return LIB
    def nvcc(*args):
        res = subprocess.run([nvcc_path(), *NVCC_FLAGS, *args], capture_output=True, text=True)
        if res.returncode != 0:
            raise RuntimeError("nvcc failed:\n" + res.stdout + res.stderr)
        if verbose:
            print(res.stderr)

    with tempfile.TemporaryDirectory() as tmp:         # the sources side by side: the instantiations of one take over a minute
        objects = [str(Path(tmp) / (src + ".o")) for src in SOURCES]
        with ThreadPoolExecutor(len(SOURCES)) as pool:
            list(pool.map(lambda job: nvcc(*(["-Xptxas", "-v"] if verbose else []), "-c", "-o", job[1], str(CSRC / job[0])),
                          zip(SOURCES, objects)))
        nvcc("-shared", "-o", str(LIB), *objects)
    return LIB


if __name__ == "__main__":
    print(build_library(force=True, verbose=True))
