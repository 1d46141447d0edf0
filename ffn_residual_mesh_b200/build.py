"""Build ``libffnrm.so`` (the C-ABI CUDA library) in-tree for sm_100a.

    python -m ffn_residual_mesh_b200.build

nvcc cross-compiles without a GPU. The shared library links the CUDA runtime
statically, so it needs only the driver at run time.
"""
from __future__ import annotations

import os
import re
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor
from importlib import metadata
from pathlib import Path

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent
CSRC = PKG / "csrc"
LIB_DIR = PKG / "lib"
LIB = LIB_DIR / "libffnrm.so"
SOURCES = [CSRC / "ffnrm.cu", CSRC / "kv.cu", PKG / "host" / "base_producer.cpp"]
HEADERS = sorted(CSRC.glob("*.cuh")) + sorted((PKG / "host").glob("*.hpp")) + [ROOT / "include" / "ffnrm.h"]
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("nvcc not found")


INCLUDES = ["-I", str(ROOT / "include"), "-I", str(CSRC), "-I", str(PKG / "host")]


def object_path(source: Path) -> Path:
    return LIB_DIR / (source.name + ".o")


def compile_command(source: Path) -> list[str]:
    return [nvcc(), *ARCH, "-O3", "-lineinfo", "-std=c++17", "-c", "-Xcompiler", "-fPIC", "-Xcompiler", "-mavx2",
            *INCLUDES, str(source), "-o", str(object_path(source))]


def link_command(out: Path = LIB) -> list[str]:
    return [nvcc(), *ARCH, "--shared", "-Xcompiler", "-fPIC", "-cudart", "static", *(str(object_path(s)) for s in SOURCES),
            "-o", str(out)]


def included(source: Path) -> list[Path]:
    """The source and every in-tree header it reaches through quoted includes."""
    found, todo = [], [source]
    while todo:
        path = todo.pop()
        found.append(path)
        for name in re.findall(r'^#include "([^"]+)"', path.read_text(), flags=re.M):
            for folder in (path.parent, ROOT / "include", CSRC, PKG / "host"):
                if (folder / name).exists() and folder / name not in found + todo:
                    todo.append(folder / name)
                    break
    return found


# Python binding of the paged cache's calls (torch tensors in, C ABI out). It belongs to one torch and one Python, which
# the stamp beside it names; the library and the runners need neither.
BIND_SOURCE = CSRC / "kv_bind.cpp"
BIND = LIB_DIR / "ffnrm_kv_bind.so"
BIND_STAMP = LIB_DIR / "ffnrm_kv_bind.stamp"


def bind_versions() -> str | None:
    """Versions that the binding is built against; None without a torch."""
    try:
        return f"torch {metadata.version('torch')}, {sys.implementation.cache_tag}"
    except metadata.PackageNotFoundError:
        return None


def build_binding(force: bool = False, verbose: bool = False) -> Path | None:
    """The binding, or None (and a message) where there is no torch with CUDA; kvcache then says that it is missing."""
    versions = bind_versions()
    if versions is None:
        print("no torch: the Python binding of the paged cache is not built", file=sys.stderr)
        return None
    same = BIND_STAMP.exists() and BIND_STAMP.read_text() == versions
    if not force and same and not stale(BIND, [BIND_SOURCE, ROOT / "include" / "ffnrm.h"]):
        return BIND
    import torch
    if torch.version.cuda is None:
        print("torch without CUDA: the Python binding of the paged cache is not built", file=sys.stderr)
        return None
    cmd = bind_command()
    if verbose:
        print(" ".join(cmd), file=sys.stderr)
    subprocess.run(cmd, check=True)
    BIND_STAMP.write_text(versions)
    return BIND


def bind_command() -> list[str]:
    import sysconfig

    import torch
    from torch.utils import cpp_extension
    cuda = Path(nvcc()).resolve().parent.parent
    libs = Path(torch.__file__).resolve().parent / "lib"
    return [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
            f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
            *(f"-isystem{p}" for p in cpp_extension.include_paths()), f"-isystem{sysconfig.get_paths()['include']}",
            f"-isystem{cuda / 'include'}", *INCLUDES, str(BIND_SOURCE), "-o", str(BIND), f"-L{LIB_DIR}", "-lffnrm", f"-L{libs}",
            "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_python", "-Wl,-rpath,$ORIGIN", f"-Wl,-rpath,{libs}"]


# Drop-in runner executables (same argv / exit codes / JSON as the reference's runners),
# host C++ over the C ABI; they find libffnrm.so through an $ORIGIN-relative rpath.
HOST = PKG / "host"
BIN_DIR = PKG / "bin"
RUNNERS = ["exact_residual_cuda_runner", "exact_main_residual_cuda_runner", "exact_cpu_base_gpu_full_ffn_runner"]
HOST_HEADERS = sorted(HOST.glob("*.hpp"))


def runner_command(name: str) -> list[str]:
    return [nvcc(), *ARCH, "-O3", "-std=c++17", "-Xcompiler", "-mavx2,-pthread", "-I", str(ROOT / "include"), "-I", str(HOST),
            str(HOST / f"{name}.cpp"), "-L", str(LIB_DIR), "-lffnrm", "-Xlinker", "-rpath,$ORIGIN/../lib",
            "-o", str(BIN_DIR / name)]


def stale(target: Path = LIB, deps: list[Path] | None = None) -> bool:
    if not target.exists():
        return True
    t = target.stat().st_mtime
    return any(p.stat().st_mtime > t for p in (deps if deps is not None else SOURCES + HEADERS))


def build_runners(force: bool = False, verbose: bool = False) -> list[Path]:
    BIN_DIR.mkdir(exist_ok=True)
    out = []
    for name in RUNNERS:
        exe = BIN_DIR / name
        if force or stale(exe, [HOST / f"{name}.cpp", LIB, ROOT / "include" / "ffnrm.h", *HOST_HEADERS]):
            cmd = runner_command(name)
            if verbose:
                print(" ".join(cmd), file=sys.stderr)
            subprocess.run(cmd, check=True)
        out.append(exe)
    return out


def build(force: bool = False, verbose: bool = False, runners: bool = True) -> Path:
    if force or stale():
        LIB_DIR.mkdir(exist_ok=True)
        todo = [compile_command(s) for s in SOURCES if force or stale(object_path(s), included(s))]
        if verbose:
            for cmd in [*todo, link_command()]:
                print(" ".join(cmd), file=sys.stderr)
        with ThreadPoolExecutor(len(SOURCES)) as pool:
            for done in pool.map(subprocess.run, todo):
                done.check_returncode()
        subprocess.run(link_command(), check=True)
    if runners:
        build_runners(force, verbose)
    build_binding(force, verbose)
    return LIB


if __name__ == "__main__":
    build(force="--force" in sys.argv, verbose=True)
    print(LIB)
