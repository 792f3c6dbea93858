"""Builds the in-tree C-ABI library ``rus_b200/liblmce.so`` with nvcc for sm_100a, and
``rus_b200/_host.so``, the C++ host side of the operators around the head, with g++
against torch's headers.

The library is compiled ahead of time (no JIT cache), so the built ``.so``
travels with the source tree. ``python -m rus_b200.build`` rebuilds it.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
import sysconfig
from pathlib import Path

PKG_DIR = Path(__file__).resolve().parent
CSRC = PKG_DIR / "csrc"
INCLUDE = PKG_DIR.parent / "include"
LIB_PATH = PKG_DIR / "liblmce.so"
SOURCES = [CSRC / "lmce_capi.cu"]
DEPS = SOURCES + sorted(CSRC.glob("*.cuh")) + [INCLUDE / "lmce.h"]
HOST_PATH = PKG_DIR / "_host.so"
HOST_DEPS = [CSRC / "lmce_host.cpp", INCLUDE / "lmce.h"]
HOST_ABI = PKG_DIR / "_host.abi"  # what _host.so was built against

ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]


def nvcc_path() -> str:
    cand = os.environ.get("NVCC") or shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not Path(cand).exists():
        raise RuntimeError("nvcc not found; set NVCC or put the CUDA toolkit on PATH")
    return cand


def compile_command(out: Path = LIB_PATH, extra: list[str] | None = None) -> list[str]:
    return [
        nvcc_path(),
        *ARCH_FLAGS,
        "-O3",
        "-lineinfo",
        "-std=c++17",
        "-shared",
        "-Xcompiler",
        "-fPIC,-fvisibility=hidden",
        "-cudart",
        "static",
        "-I",
        str(INCLUDE),
        *(extra or []),
        "-o",
        str(out),
        *[str(s) for s in SOURCES],
    ]


def host_command(out: Path = HOST_PATH) -> list[str]:
    import torch

    root = Path(torch.__file__).resolve().parent
    cuda = Path(nvcc_path()).resolve().parent.parent
    includes = [INCLUDE, root / "include", root / "include" / "torch" / "csrc" / "api" / "include", cuda / "include",
                sysconfig.get_paths()["include"]]
    return [
        os.environ.get("CXX") or "g++",
        "-O2",
        "-std=c++17",
        "-shared",
        "-fPIC",
        "-fvisibility=hidden",
        f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
        *[f"-I{p}" for p in includes],
        str(CSRC / "lmce_host.cpp"),
        "-o",
        str(out),
        f"-L{root / 'lib'}",
        "-ltorch",
        "-ltorch_cpu",
        "-lc10",
        "-lc10_cuda",
        "-ltorch_python",
        "-ldl",
    ]


def needs_build(out: Path = LIB_PATH, deps: list[Path] = DEPS) -> bool:
    if not out.exists():
        return True
    mtime = out.stat().st_mtime
    return any(dep.stat().st_mtime > mtime for dep in deps)


def host_abi() -> str:
    """What _host.so is tied to: the installed torch and the interpreter."""
    import torch

    return f"torch {torch.__version__}, {sys.implementation.cache_tag}, {sysconfig.get_platform()}\n"


def host_needs_build() -> bool:
    return (needs_build(HOST_PATH, HOST_DEPS) or not HOST_ABI.exists()
            or HOST_ABI.read_text(encoding="utf-8") != host_abi())


def build_library(force: bool = False, verbose: bool = False) -> Path:
    """Compile liblmce.so and _host.so where they are missing or older than their sources, and
    _host.so where it was built for another torch or interpreter."""
    for out, stale, command in ((LIB_PATH, lambda: needs_build(LIB_PATH), compile_command),
                                (HOST_PATH, host_needs_build, host_command)):
        if not force and not stale():
            continue
        cmd = command()
        if verbose:
            print(" ".join(cmd), flush=True)
        tmp = out.with_suffix(".so.tmp")
        cmd[cmd.index("-o") + 1] = str(tmp)
        subprocess.run(cmd, check=True)
        os.replace(tmp, out)
        if out == HOST_PATH:
            HOST_ABI.write_text(host_abi(), encoding="utf-8")
    return LIB_PATH


if __name__ == "__main__":
    build_library(force="--force" in sys.argv, verbose=True)
    print(LIB_PATH)
