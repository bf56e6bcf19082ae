"""Builds libpq_b200.so in-tree with nvcc for sm_100a (cross-compiles without a GPU), and the CPython module _bind.so that calls it
for the operators whose eager call costs more than their kernels.

    python -m pyraquant_b200.build [--force] [--verbose]
"""
from __future__ import annotations

import argparse
import hashlib
import os
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PKG = Path(__file__).resolve().parent
CSRC = PKG / "csrc"
OBJ = PKG / "csrc" / "build"
LIB = PKG / "libpq_b200.so"
BIND = PKG / "_bind.so"
SOURCES = ["api.cu", "quant.cu", "adaln_quant.cu", "gemm.cu", "gemm_lr_tc.cu", "gemm_2cta.cu", "gemm_g32.cu", "scatter.cu", "unpack4.cu", "lowrank.cu", "quant_down.cu", "linear.cu", "noalloc.cu", "quant_fp4.cu", "gemm_fp4.cu", "gemm_fp4_pair.cu", "group_norm.cu"]
NVCC_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17",
              "-Xcompiler", "-fPIC"]


def _nvcc() -> str:
    exe = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(exe):
        raise RuntimeError("nvcc not found: libpq_b200.so cannot be built")
    return exe


def _digest(paths) -> str:
    h = hashlib.sha256()
    for p in sorted(paths):
        h.update(p.name.encode())
        h.update(p.read_bytes())
    h.update(" ".join(NVCC_FLAGS).encode())
    return h.hexdigest()


def build_bind(force: bool = False, verbose: bool = False) -> Path:
    """Compiles csrc/bind.cpp against the installed torch and Python and links it to libpq_b200.so beside it."""
    import sysconfig

    import torch
    from torch.utils.cpp_extension import include_paths, library_paths
    src = CSRC / "bind.cpp"
    flags = ["-O2", "-std=c++17", "-fPIC", "-shared", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}"]
    stamp = OBJ / "bind.stamp"
    h = hashlib.sha256(src.read_bytes())
    h.update((PKG.parent / "include" / "pq_b200.h").read_bytes())
    h.update(" ".join(flags + [torch.__version__, sys.version]).encode())
    if not force and BIND.exists() and stamp.exists() and stamp.read_text() == h.hexdigest():
        return BIND
    cuda_include = Path(_nvcc()).resolve().parent.parent / "include"
    cmd = [shutil.which("g++") or "g++", *flags, str(src), "-o", str(BIND)]
    cmd += [f"-I{d}" for d in [*include_paths(), sysconfig.get_path("include"), str(cuda_include)]]
    cmd += [f"-L{d}" for d in library_paths()] + ["-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch", "-ltorch_python"]
    cmd += [f"-L{PKG}", "-l:libpq_b200.so", "-Wl,-rpath,$ORIGIN"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if verbose or r.returncode != 0:
        sys.stderr.write(r.stdout + r.stderr)
    if r.returncode != 0:
        raise RuntimeError("g++ failed on bind.cpp")
    stamp.write_text(h.hexdigest())
    return BIND


def build(force: bool = False, verbose: bool = False) -> Path:
    srcs = [CSRC / s for s in SOURCES if (CSRC / s).exists()]
    deps = srcs + sorted(CSRC.glob("*.cuh")) + [PKG.parent / "include" / "pq_b200.h"]
    stamp = OBJ / "stamp"
    digest = _digest(deps)
    if not force and LIB.exists() and stamp.exists() and stamp.read_text() == digest:
        build_bind(force, verbose)
        return LIB
    OBJ.mkdir(parents=True, exist_ok=True)
    nvcc = _nvcc()

    def compile_one(src: Path) -> Path:
        obj = OBJ / (src.stem + ".o")
        cmd = [nvcc, *NVCC_FLAGS, "-c", str(src), "-o", str(obj)]
        if verbose:
            cmd.insert(1, "-Xptxas=-v")
        r = subprocess.run(cmd, capture_output=True, text=True)
        if verbose or r.returncode != 0:
            sys.stderr.write(r.stdout + r.stderr)
        if r.returncode != 0:
            raise RuntimeError(f"nvcc failed on {src.name}")
        return obj

    with ThreadPoolExecutor(max_workers=min(8, len(srcs))) as ex:
        objs = list(ex.map(compile_one, srcs))
    cmd = [nvcc, "-shared", "-o", str(LIB), *map(str, objs), "-lcudart_static", "-lpthread", "-ldl", "-lrt"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        sys.stderr.write(r.stdout + r.stderr)
        raise RuntimeError("link of libpq_b200.so failed")
    stamp.write_text(digest)
    build_bind(force, verbose)
    return LIB


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--verbose", action="store_true")
    a = ap.parse_args()
    print(build(a.force, a.verbose))
