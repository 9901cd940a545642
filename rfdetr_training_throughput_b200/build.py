"""Build recipe for ``librfm.so`` (sm_100a) and the ``_host`` extension:
``python -m rfdetr_training_throughput_b200.build``.

Compiles every ``csrc/*.cu`` with nvcc for ``sm_100a`` into one shared library
next to this file (in-tree, so it travels with the repository snapshot).  The
CUDA runtime is linked statically: the library carries its own runtime and
binds to the process's primary context, which it shares with torch.

``csrc/host_*.cpp`` become ``_host.so``, a Python extension on torch's C++ API
that calls the library (found next to it at run time).
"""

from __future__ import annotations

import glob
import os
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
LIB_PATH = os.path.join(HERE, "librfm.so")
HOST_PATH = os.path.join(HERE, "_host.so")
OBJECTS = os.path.join(HERE, "_build")
INCLUDE = os.path.join(ROOT, "include")
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
CXX = os.environ.get("CXX", "g++")
ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC,-O2", "--expt-relaxed-constexpr"]


def sources() -> list[str]:
    return sorted(glob.glob(os.path.join(HERE, "csrc", "*.cu")))


def host_sources() -> list[str]:
    return sorted(glob.glob(os.path.join(HERE, "csrc", "host_*.cpp")))


def _newer(target: str, inputs: list[str]) -> bool:
    return os.path.exists(target) and os.path.getmtime(target) >= max(os.path.getmtime(p) for p in inputs)


def _run(cmd: list[str], verbose: bool) -> None:
    if verbose:
        print(" ".join(cmd))
    subprocess.run(cmd, check=True)


def _compile(command, inputs: list[str], headers: list[str], force: bool, verbose: bool) -> list[str]:
    """One object per source, in parallel; those newer than their source and all headers are kept."""
    os.makedirs(OBJECTS, exist_ok=True)
    objects = [os.path.join(OBJECTS, os.path.basename(s) + ".o") for s in inputs]
    stale = [(s, o) for s, o in zip(inputs, objects) if force or not _newer(o, [s, *headers])]
    with ThreadPoolExecutor(max_workers=os.cpu_count() or 1) as pool:
        list(pool.map(lambda so: _run([*command, "-c", so[0], "-o", so[1]], verbose), stale))
    return objects


def _link(cmd: list[str], target: str, verbose: bool) -> None:
    _run([*cmd, "-o", target + ".tmp"], verbose)
    os.replace(target + ".tmp", target)


def build_host(force: bool = False, verbose: bool = False) -> str:
    """``_host.so`` from ``csrc/host_*.cpp`` with the installed torch's headers and libraries."""
    headers = glob.glob(os.path.join(HERE, "csrc", "host_*.h")) + glob.glob(os.path.join(INCLUDE, "*.h"))
    if not force and _newer(HOST_PATH, host_sources() + headers):
        return HOST_PATH
    import torch

    base = os.path.dirname(torch.__file__)
    cuda = os.path.dirname(os.path.dirname(NVCC))
    include = [os.path.join(base, "include"), os.path.join(base, "include", "torch", "csrc", "api", "include"),
               os.path.join(cuda, "include"), sysconfig.get_paths()["include"], INCLUDE]
    flags = ["-O2", "-std=c++17", "-fPIC", "-fvisibility=hidden", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
             "-DTORCH_API_INCLUDE_EXTENSION_H", "-DTORCH_EXTENSION_NAME=_host"]
    objects = _compile([CXX, *flags, *(f for i in include for f in ("-isystem" if i != INCLUDE else "-I", i))],
                       host_sources(), headers, force, verbose)
    libs = os.path.join(base, "lib")
    # the shared C++ library by its name: a toolchain whose development link to it is missing would
    # take the static one, whose stream facets clash with those that torch's libraries use
    _link([CXX, "-shared", *objects, "-L", HERE, "-l:librfm.so", "-l:libstdc++.so.6", "-L", libs, "-lc10", "-lc10_cuda", "-ltorch_cpu",
           "-ltorch_cuda", "-ltorch", "-ltorch_python", "-Wl,-rpath,$ORIGIN", f"-Wl,-rpath,{libs}"], HOST_PATH, verbose)
    return HOST_PATH


def build(force: bool = False, verbose: bool = False, extra: list[str] | None = None) -> str:
    headers = glob.glob(os.path.join(HERE, "csrc", "*.cuh")) + glob.glob(os.path.join(INCLUDE, "*.h"))
    if force or not _newer(LIB_PATH, sources() + headers):
        objects = _compile([NVCC, *ARCH_FLAGS, *FLAGS, *(extra or []), "-I", INCLUDE], sources(), headers, force,
                           verbose)
        # the static runtime's own C++ library symbols stay inside: exported, they would bind
        # process-wide (they are unique symbols) and break the stream facets of other libraries
        _link([NVCC, *ARCH_FLAGS, "-shared", *objects, "-Xlinker", "--exclude-libs,ALL"], LIB_PATH, verbose)
    build_host(force, verbose)
    return LIB_PATH


if __name__ == "__main__":
    extra = ["-Xptxas", "-v"] if "--ptxas" in sys.argv else None
    print(build(force=True, verbose=True, extra=extra))
