"""Builds the native parts of gdsllm_b200 in-tree.

* ``_build/libgdsq.so``        every CUDA kernel plus the C ABI of include/gdsq.h,
                               compiled by nvcc for sm_100a only, one object per
                               ``csrc/*.cu`` (compiled side by side).
* ``_build/gds_io_ext*.so``    the torch binding that mirrors the reference's
                               ``gdsllm.runtime.gds_io_ext`` module, linked
                               against libgdsq.so.

Both are rebuilt only when a source is newer than the product.  Run
``python -m gdsllm_b200.build`` (``--force`` to rebuild everything).
"""
from __future__ import annotations

import os
import re
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PKG = Path(__file__).resolve().parent
CSRC = PKG / "csrc"
BUILD = PKG / "_build"
INCLUDE = PKG.parent / "include"
CUDA_HOME = Path(os.environ.get("CUDA_HOME", "/usr/local/cuda"))
NVCC = str(CUDA_HOME / "bin" / "nvcc")

ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ARCH_FLAGS + [
    "-lineinfo", "-O3", "-std=c++17",
    "-Xcompiler", "-fPIC,-fvisibility=hidden",
]
LINK_FLAGS = ["-Xlinker", "--exclude-libs,ALL", "-Xlinker", "-soname=libgdsq.so"]

LIB_PATH = BUILD / "libgdsq.so"
EXT_PATH = BUILD / ("gds_io_ext" + sysconfig.get_config_var("EXT_SUFFIX"))


def _newer(target: Path, sources) -> bool:
    if not target.exists():
        return True
    t = target.stat().st_mtime
    return any(Path(s).stat().st_mtime > t for s in sources)


def _run(cmd, verbose):
    if verbose:
        print(" ".join(str(c) for c in cmd), flush=True)
    subprocess.run([str(c) for c in cmd], check=True)


def _sources(path: Path, seen=None):
    """`path` and the headers of this repository that it includes."""
    seen = set() if seen is None else seen
    if path in seen:
        return seen
    seen.add(path)
    for name in re.findall(r'^#include "([^"]+)"', path.read_text(), re.M):
        for folder in (path.parent, CSRC, INCLUDE):
            if (folder / name).exists():
                _sources(folder / name, seen)
                break
    return seen


def build_lib(force: bool = False, verbose: bool = True) -> Path:
    BUILD.mkdir(parents=True, exist_ok=True)
    units = [(src, BUILD / (src.stem + ".o")) for src in sorted(CSRC.glob("*.cu"))]
    stale = [(src, obj) for src, obj in units if force or _newer(obj, _sources(src))]

    def compile_unit(unit):
        src, obj = unit
        tmp = obj.with_suffix(".o.tmp")
        _run([NVCC, *NVCC_FLAGS, "-I", INCLUDE, "-I", CSRC, "-c", "-o", tmp, src], verbose)
        os.replace(tmp, obj)

    with ThreadPoolExecutor(max_workers=4) as pool:
        list(pool.map(compile_unit, stale))
    if stale or _newer(LIB_PATH, [obj for _, obj in units]):
        tmp = LIB_PATH.with_suffix(".so.tmp")
        _run([NVCC, *ARCH_FLAGS, *LINK_FLAGS, "-shared", "-o", tmp, *[obj for _, obj in units]], verbose)
        os.replace(tmp, LIB_PATH)
    return LIB_PATH


def build_ext(force: bool = False, verbose: bool = True) -> Path:
    import torch
    from torch.utils import cpp_extension

    units = [(CSRC / name, BUILD / (Path(name).stem + ".o")) for name in ("gds_io_ext.cpp", "serve_ext.cpp")]
    stale = [(src, obj) for src, obj in units if force or _newer(obj, _sources(src))]
    if not stale and not _newer(EXT_PATH, [LIB_PATH, *[obj for _, obj in units]]):
        return EXT_PATH
    BUILD.mkdir(parents=True, exist_ok=True)
    abi = int(torch._C._GLIBCXX_USE_CXX11_ABI)
    includes = []
    for p in cpp_extension.include_paths():
        includes += ["-I", p]
    includes += ["-I", str(CUDA_HOME / "include"), "-I", sysconfig.get_paths()["include"],
                 "-I", str(INCLUDE)]

    def compile_unit(unit):
        src, obj = unit
        tmp = obj.with_suffix(".o.tmp")
        _run(["g++", "-O2", "-std=c++17", "-fPIC", "-fvisibility=hidden",
              "-DTORCH_EXTENSION_NAME=gds_io_ext", "-DTORCH_API_INCLUDE_EXTENSION_H",
              f"-D_GLIBCXX_USE_CXX11_ABI={abi}", *includes, "-c", str(src), "-o", str(tmp)], verbose)
        os.replace(tmp, obj)

    with ThreadPoolExecutor(max_workers=4) as pool:
        list(pool.map(compile_unit, stale))
    torch_lib = str(Path(torch.__file__).parent / "lib")
    tmp = EXT_PATH.with_suffix(".tmp")
    cmd = ["g++", "-shared", *[str(obj) for _, obj in units], "-o", str(tmp),
           f"-L{torch_lib}", "-lc10", "-lc10_cuda", "-ltorch", "-ltorch_cpu", "-ltorch_cuda",
           "-ltorch_python", f"-L{BUILD}", "-lgdsq", "-Wl,-rpath,$ORIGIN",
           f"-L{CUDA_HOME / 'lib64'}", "-lcudart", "-ldl"]
    _run(cmd, verbose)
    os.replace(tmp, EXT_PATH)
    return EXT_PATH


def build_all(force: bool = False, verbose: bool = True) -> None:
    build_lib(force, verbose)
    build_ext(force, verbose)


if __name__ == "__main__":
    build_all(force="--force" in sys.argv)
