"""Build recipe for liblighthouse_b200.so (sm_100a only).

Compiles every ``csrc/*.cu`` with nvcc for ``arch=compute_100a,code=sm_100a``
into objects under ``_build/`` and links them into
``liblighthouse_b200.so`` next to this file (in-tree, so the library travels
with the repository snapshot), and ``csrc/eager.cpp`` with g++ into ``_eager.so``,
the eager calls of the norm and the losses with their autograd nodes (against the
installed torch).  Rebuilds only what changed.
"""
from __future__ import annotations

import concurrent.futures as cf
import os
import pathlib
import subprocess

PKG = pathlib.Path(__file__).resolve().parent
CSRC = PKG / "csrc"
OBJ = PKG / "_build"
LIB = PKG / "liblighthouse_b200.so"
EAGER = PKG / "_eager.so"
INCLUDE = PKG.parent / "include"
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC", "-I", str(INCLUDE)]


def _headers_mtime() -> float:
    hs = list(CSRC.glob("*.cuh")) + list(INCLUDE.glob("*.h"))
    return max((h.stat().st_mtime for h in hs), default=0.0)


def _compile(src: pathlib.Path, verbose: bool) -> pathlib.Path:
    obj = OBJ / (src.stem + ".o")
    if obj.exists() and obj.stat().st_mtime >= max(src.stat().st_mtime, _headers_mtime()):
        return obj
    cmd = [NVCC, *ARCH, *FLAGS, "-c", str(src), "-o", str(obj)]
    if verbose:
        cmd.insert(1, "-Xptxas=-v")
    subprocess.run(cmd, check=True)
    return obj


def build_eager() -> pathlib.Path:
    src = CSRC / "eager.cpp"
    if EAGER.exists() and EAGER.stat().st_mtime >= max(src.stat().st_mtime, _headers_mtime()):
        return EAGER
    import sysconfig

    import torch
    from torch.utils import cpp_extension
    incs = [*cpp_extension.include_paths("cuda"), sysconfig.get_paths()["include"]]
    subprocess.run([os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared", "-DTORCH_EXTENSION_NAME=_eager",
                    "-DTORCH_API_INCLUDE_EXTENSION_H", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}",
                    *[f"-isystem{i}" for i in incs], str(src), "-o", str(EAGER),
                    *[f"-L{p}" for p in cpp_extension.library_paths()], "-lc10", "-lc10_cuda", "-ltorch_cpu",
                    "-ltorch_cuda", "-ltorch", "-ltorch_python"], check=True)
    return EAGER


def build(verbose: bool = False) -> pathlib.Path:
    OBJ.mkdir(exist_ok=True)
    srcs = sorted(CSRC.glob("*.cu"))
    with cf.ThreadPoolExecutor(max_workers=min(8, len(srcs)) + 1) as ex:
        eager = ex.submit(build_eager)
        objs = list(ex.map(lambda s: _compile(s, verbose), srcs))
        eager.result()
    if not LIB.exists() or LIB.stat().st_mtime < max(o.stat().st_mtime for o in objs):
        subprocess.run([NVCC, *ARCH, "-shared", "-o", str(LIB), *map(str, objs), "-lcudart"], check=True)
    return LIB


if __name__ == "__main__":
    import sys
    print(build(verbose="-v" in sys.argv))
