"""Build libkda.so (all CUDA kernels + the C ABI) in-tree for sm_100a.

    python kda-for-trainium_b200/build.py [-v] [--force] [-j N]

Each ``csrc/*.cu`` is compiled separately (in parallel, skipped when up to
date) into ``_build/`` and linked with the static CUDA runtime into
``kda/libkda.so``; ``csrc/binding.cpp`` (the local-attention operators' native
Python binding, against the installed torch) becomes ``kda/_binding.so``.
Without torch the library alone is built, for callers of the C ABI.  The library
does not link libcuda: the driver entry point it needs
(``cuTensorMapEncodeTiled``) is resolved at run time, so the library loads --
and its symbols can be inspected -- on a machine without a GPU.
"""

from __future__ import annotations

import argparse
import os
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path
from typing import Optional

PKG = Path(__file__).resolve().parent
REPO = PKG.parent
CSRC = PKG / "csrc"
INCLUDE = REPO / "include"
BUILD = REPO / "_build"
LIB = PKG / "kda" / "libkda.so"
BINDING = PKG / "kda" / "_binding.so"

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ARCH + [
    "-O3", "-lineinfo", "-std=c++17", "--expt-relaxed-constexpr",
    "-Xcompiler", "-fPIC,-O2", "-I", str(INCLUDE), "-I", str(CSRC),
]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("nvcc not found")


def _deps_mtime() -> float:
    hdrs = list(CSRC.glob("*.cuh")) + list(INCLUDE.glob("*.h"))
    return max((p.stat().st_mtime for p in hdrs), default=0.0)


def _compile(src: Path, force: bool, verbose: bool, extra) -> Path:
    obj = BUILD / (src.stem + ".o")
    if not force and obj.exists() and obj.stat().st_mtime >= max(src.stat().st_mtime, _deps_mtime()):
        return obj
    cmd = [nvcc(), *NVCC_FLAGS, *extra, "-c", str(src), "-o", str(obj)]
    if verbose:
        print(" ".join(cmd), flush=True)
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"nvcc failed for {src.name}:\n{r.stdout}\n{r.stderr}")
    if verbose and (r.stdout.strip() or r.stderr.strip()):
        print(r.stdout, r.stderr, flush=True)
    return obj


def _build_binding(force: bool, verbose: bool) -> Optional[Path]:
    """kda/_binding.so: host code only, resolved against the libkda.so beside it;
    None where there is no torch to build it against."""
    import importlib.util
    import sysconfig

    if importlib.util.find_spec("torch") is None:
        print("torch is not installed: kda/_binding.so (the local-attention operators in Python) is not built",
              file=sys.stderr)
        return None
    import torch
    from torch.utils.cpp_extension import include_paths, library_paths

    src = CSRC / "binding.cpp"
    stamp = BUILD / "binding.torch"  # the torch it was compiled against
    newest = max(src.stat().st_mtime, (INCLUDE / "kda.h").stat().st_mtime)
    if (not force and BINDING.exists() and BINDING.stat().st_mtime >= newest and stamp.exists()
            and stamp.read_text() == torch.__version__):
        return BINDING
    cuda_inc = Path(nvcc()).resolve().parent.parent / "include"
    inc = [*include_paths(), str(cuda_inc), sysconfig.get_paths()["include"], str(INCLUDE)]
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", str(src), "-o", str(BINDING),
           *(f"-I{p}" for p in inc), *(f"-L{p}" for p in library_paths()), "-ltorch", "-ltorch_cpu", "-ltorch_cuda", "-ltorch_python",
           "-lc10", "-lc10_cuda", f"-L{LIB.parent}", "-l:libkda.so", "-Wl,-rpath,$ORIGIN"]
    if verbose:
        print(" ".join(cmd), flush=True)
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"g++ failed for {src.name}:\n{r.stdout}\n{r.stderr}")
    stamp.write_text(torch.__version__)
    return BINDING


def build(verbose: bool = False, force: bool = False, jobs: int = 0, extra=()) -> Path:
    BUILD.mkdir(exist_ok=True)
    srcs = sorted(CSRC.glob("*.cu"))
    jobs = jobs or min(len(srcs), os.cpu_count() or 4)
    with ThreadPoolExecutor(max_workers=jobs) as ex:
        objs = list(ex.map(lambda s: _compile(s, force, verbose, list(extra)), srcs))
    newest = max(o.stat().st_mtime for o in objs)
    if force or not LIB.exists() or LIB.stat().st_mtime < newest:
        cmd = [nvcc(), *ARCH, "-shared", "-cudart", "static", "-o", str(LIB), *map(str, objs),
               "-Xlinker", "-soname=libkda.so", "-Xlinker", "--no-undefined", "-lrt", "-ldl", "-lpthread"]
        if verbose:
            print(" ".join(cmd), flush=True)
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
    _build_binding(force, verbose)
    return LIB


def main() -> int:
    ap = argparse.ArgumentParser()
    ap.add_argument("-v", "--verbose", action="store_true")
    ap.add_argument("--force", action="store_true")
    ap.add_argument("-j", "--jobs", type=int, default=0)
    ap.add_argument("--ptxas-v", action="store_true", help="print register / smem usage per kernel")
    a = ap.parse_args()
    extra = ["-Xptxas", "-v"] if a.ptxas_v else []
    lib = build(verbose=a.verbose or a.ptxas_v, force=a.force or a.ptxas_v, jobs=a.jobs, extra=extra)
    print(lib)
    return 0


if __name__ == "__main__":
    sys.exit(main())
