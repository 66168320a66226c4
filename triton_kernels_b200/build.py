"""Builds libfluxb200.so (the C-ABI library of sm_100a kernels) in-tree with nvcc, and _binding.so
(the Python binding of the operators that bind through torch's C++ API) with the host compiler.

Run as ``python -m triton_kernels_b200.build`` or call :func:`build`.  Objects are compiled
in parallel, one per ``csrc/*.cu`` file, and linked into ``triton_kernels_b200/libfluxb200.so``.
A source file is recompiled only when it (or a header) is newer than its object; the binding also
when torch's version changes.
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
INCLUDE = PKG_DIR.parent / "include"
BUILD_DIR = PKG_DIR / "build"
LIB_PATH = PKG_DIR / "libfluxb200.so"
BINDING_PATH = PKG_DIR / "_binding.so"

NVCC_FLAGS = [
    "-std=c++17",
    "-O3",
    "-gencode",
    "arch=compute_100a,code=sm_100a",
    "-lineinfo",
    "-Xcompiler",
    "-fPIC",
    "-Xptxas",
    "-v",
]


def _nvcc() -> str:
    exe = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(exe):
        raise RuntimeError("nvcc not found; the CUDA extension cannot be built")
    return exe


def _stale(target: Path, deps: list[Path]) -> bool:
    if not target.exists():
        return True
    t = target.stat().st_mtime
    return any(d.stat().st_mtime > t for d in deps)


def build(verbose: bool = False, force: bool = False) -> Path:
    """Compile every csrc/*.cu for sm_100a and link the shared library.  Returns its path."""
    nvcc = _nvcc()
    BUILD_DIR.mkdir(exist_ok=True)
    sources = sorted(CSRC.glob("*.cu"))
    headers = sorted(CSRC.glob("*.cuh")) + sorted(INCLUDE.glob("*.h"))
    jobs = []
    objects = []
    for src in sources:
        obj = BUILD_DIR / (src.stem + ".o")
        objects.append(obj)
        if force or _stale(obj, [src] + headers):
            cmd = [nvcc, *NVCC_FLAGS, "-I", str(INCLUDE), "-I", str(CSRC), "-c", str(src), "-o", str(obj)]
            jobs.append((src, cmd))

    def run(job):
        src, cmd = job
        r = subprocess.run(cmd, capture_output=True, text=True)
        (BUILD_DIR / (src.stem + ".log")).write_text(r.stdout + r.stderr)
        return src, r

    if jobs:
        with ThreadPoolExecutor(max_workers=min(8, len(jobs))) as ex:
            for src, r in ex.map(run, jobs):
                if verbose or r.returncode != 0:
                    sys.stderr.write(f"--- nvcc {src.name}\n{r.stdout}{r.stderr}\n")
                if r.returncode != 0:
                    raise RuntimeError(f"nvcc failed on {src.name}")
    if jobs or force or _stale(LIB_PATH, objects):
        cmd = [nvcc, "-shared", "-o", str(LIB_PATH), *map(str, objects), "-cudart", "static"]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            sys.stderr.write(r.stdout + r.stderr)
            raise RuntimeError("linking libfluxb200.so failed")
    build_binding(verbose, force)
    return LIB_PATH


def build_binding(verbose: bool = False, force: bool = False) -> Path:
    """Compile csrc/torch_binding.cpp against the installed torch and link it to libfluxb200.so.
    Returns its path."""
    import sysconfig

    import torch

    src = CSRC / "torch_binding.cpp"
    stamp = BUILD_DIR / "torch_binding.version"
    version = f"{torch.__version__} {sys.version_info[:2]}"
    current = stamp.exists() and stamp.read_text() == version
    if not force and current and not _stale(BINDING_PATH, [src, *INCLUDE.glob("*.h")]):
        return BINDING_PATH
    torch_dir = Path(torch.__file__).parent
    includes = [torch_dir / "include", torch_dir / "include" / "torch" / "csrc" / "api" / "include",
                sysconfig.get_paths()["include"], Path(_nvcc()).parent.parent / "include", INCLUDE]
    cmd = [
        shutil.which("g++") or "g++", "-std=c++17", "-O2", "-fPIC", "-shared", "-DTORCH_EXTENSION_NAME=_binding",
        f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", *(f"-I{p}" for p in includes), str(src),
        "-o", str(BINDING_PATH), f"-L{PKG_DIR}", "-l:libfluxb200.so", f"-L{torch_dir / 'lib'}", "-ltorch_python", "-ltorch", "-ltorch_cpu",
        "-lc10", "-lc10_cuda", "-Wl,-rpath,$ORIGIN",
    ]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if verbose or r.returncode != 0:
        sys.stderr.write(f"--- g++ {src.name}\n{r.stdout}{r.stderr}\n")
    if r.returncode != 0:
        raise RuntimeError(f"g++ failed on {src.name}")
    stamp.write_text(version)
    return BINDING_PATH


if __name__ == "__main__":
    path = build(verbose="-v" in sys.argv, force="-f" in sys.argv)
    print(path)
