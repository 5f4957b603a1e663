"""Build libfvq.so (the C-ABI CUDA library) and _fvq_torch.so (torch's short path to it) in-tree.

    python flashvsr-optimizations_b200/build.py [--force] [--verbose]

Each .cu file is compiled separately (nvcc -c, cached by mtime) and linked
into ``libfvq.so`` beside this file.  cudart is linked statically so the
library works inside any process that already has a CUDA context (torch's
included) without depending on which libcudart that process loaded.
``_fvq_torch.so`` is host code only, compiled against the installed torch (and
left out where there is none).
"""
from __future__ import annotations

import argparse
import os
import shutil
import subprocess
import sys
from pathlib import Path

HERE = Path(__file__).resolve().parent
CSRC = HERE / "csrc"
INCLUDE = HERE.parent / "include"
BUILD = HERE / "_build"
LIB = HERE / "libfvq.so"
BINDING = HERE / "_fvq_torch.so"

SOURCES = ["fvq_quant.cu", "fvq_fp8.cu", "fvq_resize.cu", "fvq_block.cu", "fvq_gemm.cu",
           "fvq_norm.cu", "fvq_linear.cu", "fvq_cache.cu", "fvq_api.cu", "fvq_noalloc.cu"]
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ARCH + [
    "-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC,-O2",
    "--expt-relaxed-constexpr", "-Xptxas", "-v",
    f"-I{INCLUDE}", f"-I{CSRC}",
]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", shutil.which("nvcc")):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("nvcc not found (set NVCC or install the CUDA toolkit)")


def _headers_mtime() -> float:
    hs = list(CSRC.glob("*.cuh")) + list(CSRC.glob("*.h")) + list(INCLUDE.glob("*.h"))
    return max((h.stat().st_mtime for h in hs), default=0.0)


def build(force: bool = False, verbose: bool = False) -> Path:
    BUILD.mkdir(exist_ok=True)
    hdr = _headers_mtime()
    objs = []
    changed = force or not LIB.exists()
    for src in SOURCES:
        s = CSRC / src
        o = BUILD / (src + ".o")
        objs.append(o)
        if force or not o.exists() or o.stat().st_mtime < max(s.stat().st_mtime, hdr):
            cmd = [nvcc(), *NVCC_FLAGS, "-c", str(s), "-o", str(o)]
            res = subprocess.run(cmd, capture_output=True, text=True)
            if verbose or res.returncode != 0:
                sys.stderr.write(res.stdout + res.stderr)
            if res.returncode != 0:
                raise RuntimeError(f"nvcc failed on {src}")
            (BUILD / (src + ".ptxas.txt")).write_text(res.stderr)
            changed = True
    if changed or any(o.stat().st_mtime > LIB.stat().st_mtime for o in objs):
        tmp = LIB.with_suffix(".so.tmp")
        cmd = [nvcc(), *ARCH, "-shared", "-cudart", "static", "-o", str(tmp), *map(str, objs)]
        res = subprocess.run(cmd, capture_output=True, text=True)
        if res.returncode != 0:
            sys.stderr.write(res.stdout + res.stderr)
            raise RuntimeError("link of libfvq.so failed")
        os.replace(tmp, LIB)
    return LIB


def build_binding(force: bool = False) -> Path:
    """_fvq_torch.so, rebuilt when its source, the C header or the installed torch changed."""
    import sysconfig

    import torch
    src = CSRC / "fvq_torch.cpp"
    stamp = BUILD / "fvq_torch.version.txt"
    version = f"{torch.__version__} {sys.version}"
    newest = max(src.stat().st_mtime, max(h.stat().st_mtime for h in INCLUDE.glob("*.h")))
    if not force and BINDING.exists() and BINDING.stat().st_mtime >= newest and stamp.exists() \
            and stamp.read_text() == version:
        return BINDING
    BUILD.mkdir(exist_ok=True)
    root = Path(torch.__file__).resolve().parent
    cuda = Path(nvcc()).resolve().parent.parent / "include"
    tmp = BINDING.with_suffix(".so.tmp")
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           *(f"-isystem{p}" for p in (root / "include", root / "include/torch/csrc/api/include",
                                      sysconfig.get_paths()["include"], cuda)),
           str(src), "-o", str(tmp), f"-L{root / 'lib'}", "-ltorch_python", "-ltorch_cpu", "-ltorch_cuda",
           "-lc10", "-lc10_cuda"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        sys.stderr.write(res.stdout + res.stderr)
        raise RuntimeError("build of _fvq_torch.so failed")
    os.replace(tmp, BINDING)
    stamp.write_text(version)
    return BINDING


def main(argv: list[str] | None = None) -> None:
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--verbose", action="store_true")
    a = ap.parse_args(argv)
    print(build(a.force, a.verbose))
    try:
        print(build_binding(a.force))
    except ModuleNotFoundError as e:  # the C ABI needs no torch
        if e.name != "torch":
            raise
        print(f"{BINDING.name} not built: torch is not installed")


if __name__ == "__main__":
    main()
