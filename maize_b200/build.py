"""Builds ``maize_b200/_lib/libmaize_gemm.so`` from ``csrc/`` with nvcc for sm_100a.

Run as ``python -m maize_b200.build``.  nvcc cross-compiles without a GPU; the
library links the CUDA runtime statically and resolves the one driver symbol it
needs (``cuTensorMapEncodeTiled``) at run time, so it loads on a machine with
no driver and reports ``MAIZE_ERR_NO_DEVICE`` there instead of failing to load.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
import sysconfig
from pathlib import Path

PKG = Path(__file__).resolve().parent
CSRC = PKG / "csrc"
OUT = PKG / "_lib" / "libmaize_gemm.so"
SOURCES = [CSRC / "maize_gemm.cu", CSRC / "maize_mgpu.cu", CSRC / "maize_experts.cu",
           CSRC / "maize_e4m3.cu"]
# Python callables for the host-bound entry points, linked to the library beside it
CALLS_SOURCE = CSRC / "calls.c"
CALLS_OUT = OUT.with_name("maize_calls" + (sysconfig.get_config_var("EXT_SUFFIX") or ".so"))
HEADER = PKG.parent / "include" / "maize_gemm.h"
DEPENDS = sorted(CSRC.glob("*.cu")) + sorted(CSRC.glob("*.cuh")) + [HEADER]

NVCC_FLAGS = [
    "-std=c++17", "-O3", "-lineinfo",
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-Xcompiler", "-fPIC,-fvisibility=hidden",
    "-shared", "-cudart", "static",
]


def find_nvcc() -> str:
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not Path(nvcc).exists():
        raise RuntimeError("nvcc not found: the CUDA kernels cannot be built")
    return nvcc


def _older(target: Path, sources) -> bool:
    return not target.exists() or any(s.stat().st_mtime > target.stat().st_mtime for s in sources if s.exists())


def is_stale() -> bool:
    return _older(OUT, DEPENDS)


def _calls_compiler() -> str | None:
    """A C compiler, where Python's headers are there for it."""
    if not Path(sysconfig.get_paths()["include"], "Python.h").exists():
        return None
    return shutil.which("gcc") or shutil.which("cc")


def calls_are_stale() -> bool:
    """Whether the callables are missing or old, and this machine could build them."""
    return _calls_compiler() is not None and _older(CALLS_OUT, (CALLS_SOURCE, HEADER))


def build(force: bool = False, verbose: bool = False) -> Path:
    if force or is_stale():
        OUT.parent.mkdir(parents=True, exist_ok=True)
        cmd = [find_nvcc(), *NVCC_FLAGS, *(["-Xptxas", "-v"] if verbose else []), "-o", str(OUT), *map(str, SOURCES)]
        env = dict(os.environ)
        proc = subprocess.run(cmd, env=env, capture_output=True, text=True)
        if verbose or proc.returncode != 0:
            sys.stderr.write(proc.stdout + proc.stderr)
        if proc.returncode != 0:
            raise RuntimeError("nvcc failed building libmaize_gemm.so")
        build_calls()
    elif calls_are_stale():
        build_calls()
    return OUT


def build_calls() -> None:
    """Builds ``csrc/calls.c``.  Where Python's headers or a C compiler are missing, or the compiler fails, the binding calls
    through ctypes."""
    cc = _calls_compiler()
    if cc is None:
        sys.stderr.write("maize_b200: no C compiler or Python.h, calls go through ctypes\n")
        CALLS_OUT.unlink(missing_ok=True)
        return
    cmd = [cc, "-O2", "-Wall", "-shared", "-fPIC", f"-I{sysconfig.get_paths()['include']}", "-o", str(CALLS_OUT), str(CALLS_SOURCE),
           f"-L{OUT.parent}", f"-l:{OUT.name}", "-Wl,-rpath,$ORIGIN"]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        sys.stderr.write(proc.stdout + proc.stderr)
        sys.stderr.write("maize_b200: the C compiler failed building calls.c, calls go through ctypes\n")
        CALLS_OUT.unlink(missing_ok=True)


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
