"""Build ``libeo_b200.so`` in-tree with nvcc for sm_100a (cross-compiles without a GPU), and the Python extension
``_host-torch<version>.<python abi>.so`` (tables of tensor addresses, ``csrc/host_tables.cpp``) with g++ against the installed torch.

Usage: ``python -m emerging_optimizers_b200.build [--force] [--verbose]``
"""

from __future__ import annotations

import argparse
import os
import shutil
import subprocess
import sys
import sysconfig

import torch


PKG_DIR = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(PKG_DIR, "csrc")
OUT = os.path.join(PKG_DIR, "libeo_b200.so")
SOURCES = ["eo_b200.cu"]
HOST_SOURCE = os.path.join(CSRC, "host_tables.cpp")
NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-std=c++17", "-lineinfo",
    "-shared", "-Xcompiler", "-fPIC",
]  # fmt: skip


def host_path() -> str:
    """Path of the host extension for this torch and this Python.  Both are part of its name: a module built against another
    version has another name, so that it is neither loaded nor taken for up to date."""
    return os.path.join(PKG_DIR, f"_host-torch{torch.__version__}{sysconfig.get_config_var('EXT_SUFFIX')}")


HOST_OUT = host_path()


def _nvcc() -> str:
    exe = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(exe):
        raise RuntimeError("nvcc not found; libeo_b200.so cannot be built")
    return exe


def _inputs() -> list[str]:
    files = []
    for root in (CSRC, os.path.join(os.path.dirname(PKG_DIR), "include")):
        for name in sorted(os.listdir(root)):
            if name.endswith((".cu", ".cuh", ".h")):
                files.append(os.path.join(root, name))
    return files


def needs_build() -> bool:
    if not os.path.exists(OUT):
        return True
    built = os.path.getmtime(OUT)
    return any(os.path.getmtime(f) > built for f in _inputs())


def _run(cmd: list[str], tmp: str, out: str) -> str:
    """Run a compiler that writes ``tmp`` and move the result to ``out``: a reader never sees a half-written file."""
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        if os.path.exists(tmp):
            os.remove(tmp)
        raise RuntimeError(f"{os.path.basename(cmd[0])} failed:\n{' '.join(cmd)}\n{res.stdout}\n{res.stderr}")
    os.replace(tmp, out)
    return res.stderr


def build_host(force: bool = False) -> str:
    """Compile the host extension for this torch and Python if it is missing or its source is newer; return its path."""
    out = host_path()
    if not force and os.path.exists(out) and os.path.getmtime(HOST_SOURCE) <= os.path.getmtime(out):
        return out
    from torch.utils import cpp_extension

    cuda_home = os.path.dirname(os.path.dirname(os.path.realpath(_nvcc())))
    includes = [*cpp_extension.include_paths(), os.path.join(cuda_home, "include"), sysconfig.get_paths()["include"]]
    lib_dir = os.path.join(os.path.dirname(torch.__file__), "lib")
    tmp = f"{out}.{os.getpid()}.tmp"
    cmd = [
        shutil.which("g++") or "g++", "-O2", "-std=c++17", "-shared", "-fPIC",
        f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}",
        *[f"-I{p}" for p in includes], "-o", tmp, HOST_SOURCE,
        f"-L{lib_dir}", "-ltorch_python", "-ltorch", "-lc10", "-lc10_cuda", f"-Wl,-rpath,{lib_dir}",
    ]  # fmt: skip
    _run(cmd, tmp, out)
    return out


def build(force: bool = False, verbose: bool = False, extra_flags: list[str] | None = None) -> str:
    """Compile the library and the host extension where a source is newer; return the path of the library."""
    build_host(force)
    if not force and not needs_build():
        return OUT
    cmd = [_nvcc(), *NVCC_FLAGS, *(extra_flags or [])]
    if verbose:
        cmd += ["-Xptxas", "-v"]
    tmp = f"{OUT}.{os.getpid()}.tmp"
    cmd += ["-o", tmp, *[os.path.join(CSRC, s) for s in SOURCES]]
    messages = _run(cmd, tmp, OUT)
    if verbose:
        print(messages, file=sys.stderr)
    return OUT


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--verbose", action="store_true")
    ap.add_argument("--define", action="append", default=[])
    args = ap.parse_args()
    print(build(args.force, args.verbose, [f"-D{d}" for d in args.define]))
