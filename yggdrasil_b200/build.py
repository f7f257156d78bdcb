"""Build libygg_b200.so in-tree with nvcc for sm_100a, and _ops.so, the operators' calls on torch tensors, with the C++
compiler against torch's headers (both travel with the tree; nothing is JIT-compiled).

    python -m yggdrasil_b200.build [--verbose]
"""
from __future__ import annotations

import argparse
import os
import shutil
import subprocess
import sys
from pathlib import Path

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent
CSRC = PKG / "csrc"
LIB = PKG / "libygg_b200.so"
OPS = PKG / "_ops.so"
OPS_SOURCE = CSRC / "ygg_torch.cpp"
SOURCES = [CSRC / "ygg_load.cu", CSRC / "ygg_step.cu", CSRC / "ygg_coop.cu", CSRC / "ygg_grouped.cu",
           CSRC / "ygg_float.cu", CSRC / "ygg_logprobs.cu", CSRC / "ygg_linear.cu",
           CSRC / "ygg_pages.cu"]
HEADERS = [CSRC / "ygg_model.h", CSRC / "ygg_smem.h", CSRC / "ygg_device.cuh", CSRC / "ygg_ops.cuh",
           CSRC / "ygg_tensor.cuh", ROOT / "include" / "ygg_b200.h"]
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
# no --use_fast_math and no FMA contraction: every f32 op of the step is single-rounded as in the reference
FLAGS = ["-O3", "-std=c++17", "-lineinfo", "--fmad=false", "-Xcompiler", "-fPIC", "-cudart", "static",
         "-Xcompiler", "-fvisibility=hidden"]


def nvcc() -> str:
    for c in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if c and Path(c).exists():
            return c
    raise RuntimeError("nvcc not found")


def stale(target: Path, sources) -> bool:
    if not target.exists():
        return True
    t = target.stat().st_mtime
    return any(p.stat().st_mtime > t for p in sources)


def build(verbose: bool = False, force: bool = False) -> Path:
    """Compile what a source is newer than; returns the library's path."""
    if force or stale(LIB, SOURCES + HEADERS):
        build_library(verbose)
    if force or stale(OPS, [OPS_SOURCE, ROOT / "include" / "ygg_b200.h"]):
        build_ops()
    return LIB


def build_library(verbose: bool) -> None:
    objs, procs = [], []
    tmp = PKG / "_build"
    tmp.mkdir(exist_ok=True)
    for src in SOURCES:   # the translation units compile in parallel
        obj = tmp / (src.stem + ".o")
        cmd = [nvcc(), *ARCH, *FLAGS, "-I", str(ROOT / "include"), "-c", str(src), "-o", str(obj)]
        if verbose:
            cmd += ["-Xptxas", "-v"]
        procs.append((src, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True)))
        objs.append(str(obj))
    for src, p in procs:
        out, err = p.communicate()
        if p.returncode:
            raise RuntimeError(f"nvcc failed on {src.name}:\n{out}\n{err}")
        if verbose:
            print(err, file=sys.stderr)
    run([nvcc(), *ARCH, "-shared", "-cudart", "static", "-o", str(LIB), *objs], "link")


def build_ops() -> None:
    import sysconfig

    import torch
    home = Path(torch.__file__).resolve().parent
    cuda = Path(nvcc()).resolve().parents[1] / "include"
    abi = int(torch._C._GLIBCXX_USE_CXX11_ABI)
    system = [x for d in (home / "include", home / "include" / "torch" / "csrc" / "api" / "include", cuda)
              for x in ("-isystem", str(d))]
    run([os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
         f"-D_GLIBCXX_USE_CXX11_ABI={abi}", "-I", str(ROOT / "include"), "-I", sysconfig.get_paths()["include"], *system,
         str(OPS_SOURCE), "-o", str(OPS), "-L", str(home / "lib"), "-ltorch_python", "-ltorch_cuda", "-ltorch_cpu",
         "-lc10_cuda", "-lc10", "-L", str(PKG), "-l:" + LIB.name, "-Wl,-rpath,$ORIGIN"], "the torch binding")


def run(cmd, what: str) -> None:
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode:
        raise RuntimeError(f"{what} failed:\n{r.stdout}\n{r.stderr}")


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--verbose", action="store_true")
    ap.add_argument("--force", action="store_true")
    a = ap.parse_args()
    print(build(a.verbose, a.force))
