"""Builds libb200kernels.so in-tree with nvcc for sm_100a, and the extension module _tensor_list.so with g++ against torch's headers.

Usage: ``python -m triton_tenstorrent_b200.build [--force] [--verbose]``.
The library sits next to this file so that it travels with the source tree; nothing is
installed into site-packages and nothing is JIT-compiled at import time.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PKG_DIR = Path(__file__).resolve().parent
CSRC = PKG_DIR / "csrc"
LIB_PATH = PKG_DIR / "libb200kernels.so"
TENSOR_LIST_PATH = PKG_DIR / "_tensor_list.so"
BUILD_DIR = PKG_DIR / "build"

SOURCES = ["capi.cu", "elementwise.cu", "matmul_tcgen05.cu", "attn_fwd_tcgen05.cu", "attn_bwd_tcgen05.cu", "layer_norm.cu", "lce_tcgen05.cu",
           "adamw.cu", "selftest.cu"]

NVCC_FLAGS = [
    "-std=c++17",
    "-O3",
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-lineinfo",
    "-Xcompiler", "-fPIC",
    "--expt-relaxed-constexpr",
]


def _nvcc() -> str:
    cand = os.environ.get("NVCC") or shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not Path(cand).exists():
        raise RuntimeError("nvcc not found; set NVCC or put it on PATH")
    return cand


def _stale(target: Path, deps) -> bool:
    if not target.exists():
        return True
    t = target.stat().st_mtime
    return any(Path(d).stat().st_mtime > t for d in deps)


def _tensor_list_command(source: Path):
    """The command that compiles and links the extension module; torch's libraries are those that the process has loaded already."""
    import sysconfig

    import torch

    root = Path(torch.__file__).resolve().parent
    include = [root / "include", root / "include" / "torch" / "csrc" / "api" / "include", sysconfig.get_paths()["include"], PKG_DIR.parent / "include",
               Path(_nvcc()).resolve().parent.parent / "include"]
    return ["g++", "-std=c++17", "-O2", "-fPIC", "-shared", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}", *(f"-I{p}" for p in include),
            f"-L{root / 'lib'}", "-Wl,--no-as-needed", "-lc10", "-ltorch_cpu", "-ltorch_python", str(source), "-o", str(TENSOR_LIST_PATH)]


def build(force: bool = False, verbose: bool = False) -> Path:
    """Compiles every .cu under csrc/ and links the shared library.  Returns its path."""
    nvcc = _nvcc()
    BUILD_DIR.mkdir(exist_ok=True)
    headers = list(CSRC.glob("*.h")) + list(CSRC.glob("*.cuh")) + [PKG_DIR.parent / "include" / "b200k.h", Path(__file__)]
    objs = []
    jobs = []
    for src in SOURCES:
        s = CSRC / src
        o = BUILD_DIR / (s.stem + ".o")
        objs.append(o)
        if force or _stale(o, [s, *headers]):
            cmd = [nvcc, *NVCC_FLAGS, "-c", str(s), "-o", str(o)]
            if verbose:
                cmd.insert(1, "-Xptxas")
                cmd.insert(2, "-v")
            jobs.append(cmd)

    tensor_list = _tensor_list_command(CSRC / "tensor_list.cpp") if force or _stale(TENSOR_LIST_PATH, [CSRC / "tensor_list.cpp", *headers]) else None

    def run(cmd):
        r = subprocess.run(cmd, capture_output=True, text=True)
        if verbose or r.returncode != 0:
            sys.stderr.write(" ".join(cmd) + "\n" + r.stdout + r.stderr)
        if r.returncode != 0:
            raise RuntimeError(f"{Path(cmd[0]).name} failed on {cmd[-3]}")

    if jobs or tensor_list:
        with ThreadPoolExecutor(max_workers=min(4, len(jobs) + 1)) as ex:
            list(ex.map(run, jobs + ([tensor_list] if tensor_list else [])))
    if jobs or force or _stale(LIB_PATH, objs):
        link = [nvcc, "-shared", "-o", str(LIB_PATH), *map(str, objs), "-gencode", "arch=compute_100a,code=sm_100a"]
        run(link)
    return LIB_PATH


if __name__ == "__main__":
    path = build(force="--force" in sys.argv, verbose="--verbose" in sys.argv)
    print(path)
