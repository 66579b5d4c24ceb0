"""Build the native libraries of the MoE FFN grouped-GEMM path in-tree.

Outputs (git-ignored, shipped with the source tree):
  cutlass_op/bf16_grouped_mm/libmoe_gemm.so        C ABI (include/moe_gemm.h), sm_100a kernels
  cutlass_op/bf16_grouped_mm/_grouped_mm_ops.so    torch.library ops `grouped_mm::*` over that ABI

Only nvcc (for sm_100a) and g++ are used; no JIT cache outside the tree.  Every source is compiled to
an object under _build/ (git-ignored), several at a time; an object is rebuilt when its source or any
header is newer, a library when any of its objects is.
"""

from __future__ import annotations

import os
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PKG_ROOT = Path(__file__).resolve().parent
REPO_ROOT = PKG_ROOT.parent
CSRC = PKG_ROOT / "csrc"
INCLUDE = REPO_ROOT / "include"
OUT_DIR = PKG_ROOT / "cutlass_op" / "bf16_grouped_mm"
LIB = OUT_DIR / "libmoe_gemm.so"
OPS = OUT_DIR / "_grouped_mm_ops.so"
OBJ_DIR = PKG_ROOT / "_build"

CUDA_HOME = Path(os.environ.get("CUDA_HOME", "/usr/local/cuda"))
NVCC = CUDA_HOME / "bin" / "nvcc"
ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]


def _newer(target: Path, deps: list[Path]) -> bool:
    if not target.exists():
        return True
    t = target.stat().st_mtime
    return any(d.stat().st_mtime > t for d in deps)


def _run(cmd: list[str], verbose: bool) -> None:
    if verbose:
        print(" ".join(str(c) for c in cmd), flush=True)
    subprocess.run([str(c) for c in cmd], check=True)


def _objects(srcs: list[Path], headers: list[Path], cmd: list, verbose: bool, force: bool) -> list[Path]:
    """Compile every source that is out of date (`cmd` + -c source -o object); the objects' paths."""
    OBJ_DIR.mkdir(exist_ok=True)
    objs = [OBJ_DIR / f"{s.stem}.o" for s in srcs]
    todo = [(s, o) for s, o in zip(srcs, objs) if force or _newer(o, [s, *headers])]
    with ThreadPoolExecutor(max_workers=max(1, os.cpu_count() or 1)) as pool:
        list(pool.map(lambda so: _run([*cmd, "-c", so[0], "-o", so[1]], verbose), todo))
    return objs


def build_lib(verbose: bool = False, force: bool = False) -> Path:
    headers = sorted(CSRC.glob("*.cuh")) + sorted(CSRC.glob("*.h")) + sorted(INCLUDE.glob("*.h"))
    cmd = [NVCC, *ARCH_FLAGS, "-O3", "-lineinfo", "-std=c++17", "--expt-relaxed-constexpr", "-Xcompiler", "-fPIC",
           f"-I{INCLUDE}", f"-I{CSRC}"]
    objs = _objects(sorted(CSRC.glob("*.cu")), headers, cmd, verbose, force)
    if force or _newer(LIB, objs):
        _run([NVCC, *ARCH_FLAGS, "-shared", "-o", LIB, *objs], verbose)
    return LIB


def build_ops(verbose: bool = False, force: bool = False) -> Path:
    import torch
    import torch.utils.cpp_extension as ext

    libdirs = ext.library_paths(device_type="cuda")
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           "-DTORCH_API_INCLUDE_EXTENSION_H", *[f"-I{p}" for p in ext.include_paths(device_type="cuda")],
           f"-I{INCLUDE}"]
    objs = _objects(sorted(CSRC.glob("torch_ops*.cpp")), sorted(INCLUDE.glob("*.h")), cmd, verbose, force)
    if force or _newer(OPS, [*objs, LIB]):
        _run(["g++", "-shared", *objs, "-o", OPS, *[f"-L{d}" for d in libdirs], f"-L{OUT_DIR}",
              "-lmoe_gemm", "-lc10", "-lc10_cuda", "-ltorch", "-ltorch_cpu", "-ltorch_cuda", "-lcudart",
              "-Wl,-rpath,$ORIGIN", *[f"-Wl,-rpath,{d}" for d in libdirs]], verbose)
    return OPS


def build(verbose: bool = False, force: bool = False) -> None:
    build_lib(verbose, force)
    build_ops(verbose, force)


if __name__ == "__main__":
    build(verbose=True, force="--force" in sys.argv)
