"""Builds the sm_100a shared library of the paged-attention path in-tree.

    python -m batchstream_inference_engine_b200.build

compiles every ``csrc/*.cu`` with nvcc for ``sm_100a`` only and links
``libbatchstream_b200.so`` next to this file.  The CUDA runtime is linked
statically and its symbols are kept local to the library, so the library does
not depend on (or interfere with) the runtime that PyTorch loads; the driver is
reached at run time through the runtime's entry-point query, so the library
also loads on a machine without a GPU driver.

``csrc/binding.cpp`` becomes ``_native.so``, the Python entry points of the
bounded-cache operators: a C++ extension over torch's headers, linked against
``libbatchstream_b200.so`` (found next to it) and the libraries torch has loaded.
"""

from __future__ import annotations

import os
import shutil
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor
from importlib.metadata import version
from pathlib import Path

PACKAGE = Path(__file__).resolve().parent
CSRC = PACKAGE / "csrc"
BUILD = PACKAGE / "_build"
LIBRARY = PACKAGE / "libbatchstream_b200.so"
BINDING = PACKAGE / "_native.so"
BINDING_FOR = BUILD / "native_for.txt"  # what the extension was built against
INCLUDE = PACKAGE.parent / "include"

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
CFLAGS = ["-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC", "--expt-relaxed-constexpr"]


def nvcc() -> str:
    found = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not Path(found).exists():
        raise RuntimeError("nvcc not found: the CUDA toolkit is needed to build the library")
    return found


def _stale(target: Path, sources: list[Path]) -> bool:
    if not target.exists():
        return True
    mtime = target.stat().st_mtime
    return any(src.stat().st_mtime > mtime for src in sources)


def build(verbose: bool = False, force: bool = False) -> Path:
    """Compile (if stale) and return the path of the shared library."""
    BUILD.mkdir(exist_ok=True)
    headers = sorted(CSRC.glob("*.cuh")) + sorted(INCLUDE.glob("*.h"))
    sources = sorted(CSRC.glob("*.cu"))
    compiler = nvcc()

    def compile_one(src: Path) -> Path:
        obj = BUILD / (src.stem + ".o")
        if force or _stale(obj, [src, *headers]):
            cmd = [compiler, *ARCH, *CFLAGS, f"-I{INCLUDE}", "-c", str(src), "-o", str(obj)]
            if verbose:
                cmd.insert(1, "-Xptxas=-v")
            proc = subprocess.run(cmd, capture_output=True, text=True)
            if proc.returncode != 0:
                raise RuntimeError(f"nvcc failed on {src.name}:\n{proc.stderr}")
            if verbose and proc.stderr:
                print(proc.stderr, file=sys.stderr)
        return obj

    with ThreadPoolExecutor(max_workers=min(8, os.cpu_count() or 1)) as pool:
        objects = list(pool.map(compile_one, sources))

    if force or _stale(LIBRARY, objects):
        tmp = LIBRARY.with_suffix(".so.tmp")
        cmd = [
            compiler, *ARCH, "-shared", "-cudart", "static",
            "-Xlinker", "--exclude-libs,ALL", "-Xlinker", "-Bsymbolic",
            *[str(o) for o in objects], "-o", str(tmp),
        ]
        proc = subprocess.run(cmd, capture_output=True, text=True)
        if proc.returncode != 0:
            raise RuntimeError(f"linking libbatchstream_b200.so failed:\n{proc.stderr}")
        tmp.replace(LIBRARY)
    build_binding(force)
    return LIBRARY


def binding_against() -> str:
    """The versions of Python and torch that the extension's binary interface is tied to."""
    return f"{sys.implementation.cache_tag} torch {version('torch')}"


def build_binding(force: bool = False) -> Path:
    """Compile (if stale) and return the path of the Python extension."""
    source = CSRC / "binding.cpp"
    against = binding_against()
    if not (force or _stale(BINDING, [source, INCLUDE / "batchstream_b200.h"])
            or not BINDING_FOR.exists() or BINDING_FOR.read_text() != against):
        return BINDING
    compiler = shutil.which("g++")
    if compiler is None:
        raise RuntimeError("g++ not found: it is needed to build the Python extension")
    import torch

    root = Path(torch.__file__).resolve().parent
    cuda = Path(nvcc()).resolve().parent.parent
    tmp = BINDING.with_suffix(".so.tmp")
    cmd = [
        compiler, "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
        f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
        f"-I{INCLUDE}", f"-I{root / 'include'}",
        f"-I{root / 'include' / 'torch' / 'csrc' / 'api' / 'include'}",
        f"-I{sysconfig.get_paths()['include']}", f"-I{cuda / 'include'}",
        str(source), "-o", str(tmp), f"-L{PACKAGE}", "-lbatchstream_b200", f"-L{root / 'lib'}",
        "-ltorch_python", "-ltorch_cpu", "-lc10_cuda", "-lc10", "-Wl,-rpath,$ORIGIN",
    ]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"building {BINDING.name} failed:\n{proc.stderr}")
    tmp.replace(BINDING)
    BINDING_FOR.write_text(against)
    return BINDING


if __name__ == "__main__":
    print(build(verbose="-v" in sys.argv, force="--force" in sys.argv))
