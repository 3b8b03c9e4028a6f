"""Builds libbullet_b200.so in-tree with nvcc for sm_100a (cross-compiles without a GPU), and the module of the tensor calls (ops.py).

    python -m bullet_b200.build [--verbose]
"""
from __future__ import annotations

import importlib.metadata
import importlib.util
import os
import shutil
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libbullet_b200.so")
HEADER = os.path.join(HERE, "..", "include", "bullet_b200.h")
TENSOR_CALLS = os.path.join(HERE, "_tensor_calls.so")
MADE_FOR = os.path.join(HERE, "_tensor_calls.made_for")
SOURCES = ["net.cu", "op_ft_forward.cu", "op_rows.cu", "op_dense.cu", "op_four.cu", "op_table.cu", "op_clip.cu", "gave_up.cu", "probe.cu", "host_pack.cpp", "checkpoint.cpp", "saved_format.cpp"]


def _nvcc() -> str:
    for cand in (shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found: bullet_b200 has no CPU fallback and cannot be built without the CUDA toolkit")


def _stale(output: str, deps: list[str]) -> bool:
    return not os.path.exists(output) or any(os.path.getmtime(p) > os.path.getmtime(output) for p in deps)


def _library_sources() -> list[str]:
    """What the library is made of: all of csrc but the tensor calls."""
    return [os.path.join(CSRC, f) for f in sorted(os.listdir(CSRC)) if f != "tensor_calls.cpp"] + [HEADER]


def build(force: bool = False, verbose: bool = False) -> str:
    """Builds what is out of date.  The library needs no torch; without a module of the tensor calls only ops.py cannot be imported."""
    host_cxx = "/usr/bin/g++" if os.path.exists("/usr/bin/g++") else "g++"  # needs libgomp
    if force or _stale(LIB, _library_sources()):
        cmd = [_nvcc(), "-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17",
               "-ccbin", host_cxx, "-Xcompiler", "-fPIC,-fopenmp,-O3,-Wall", "-shared", "-o", LIB]
        if verbose:
            cmd += ["-Xptxas", "-v"]
        cmd += [os.path.join(CSRC, s) for s in SOURCES] + ["-lgomp", "-lcudart"]
        res = subprocess.run(cmd, capture_output=True, text=True)
        if verbose or res.returncode:
            sys.stderr.write(res.stdout + res.stderr)
        if res.returncode:
            raise RuntimeError("nvcc failed building libbullet_b200.so")
    if force or _tensor_calls_stale():
        build_tensor_calls(host_cxx, verbose)
    return LIB


def _torch_dir() -> str | None:
    spec = importlib.util.find_spec("torch")
    return os.path.dirname(spec.origin) if spec and spec.origin else None


def _made_for() -> str:
    """The torch and Python that the module of the tensor calls is made for; it is of no use with others."""
    try:
        version = importlib.metadata.version("torch")
    except importlib.metadata.PackageNotFoundError:
        version = "?"
    return f"torch {version} in {_torch_dir()}, {sys.implementation.cache_tag}"


def _tensor_calls_stale() -> bool:
    if _torch_dir() is None:
        return False
    if _stale(TENSOR_CALLS, [os.path.join(CSRC, "tensor_calls.cpp"), HEADER]) or not os.path.exists(MADE_FOR):
        return True
    with open(MADE_FOR) as f:
        return f.read() != _made_for()


def _tensor_calls_lack() -> str | None:
    """What the module cannot be built without and is not there."""
    torch_dir = _torch_dir()
    if torch_dir is None:
        return "torch"
    for path in (os.path.join(torch_dir, "lib", "libtorch_cuda.so"), os.path.join(torch_dir, "lib", "libc10_cuda.so"), os.path.join(torch_dir, "include", "c10", "cuda", "CUDAStream.h"),
                 os.path.join(sysconfig.get_paths()["include"], "Python.h")):
        if not os.path.exists(path):
            return path
    return None


def build_tensor_calls(host_cxx: str, verbose: bool = False) -> str | None:
    """The module behind ops.py, against the torch that is installed; None, with a message, where that cannot be: ops.py then says
    at its import that the module is missing."""
    for old in (TENSOR_CALLS, MADE_FOR):
        if os.path.exists(old):
            os.remove(old)
    lack = _tensor_calls_lack()
    if lack:
        sys.stderr.write(f"{lack} is not installed: bullet_b200.ops is not built\n")
        return None
    torch_dir = _torch_dir()
    include, lib = os.path.join(torch_dir, "include"), os.path.join(torch_dir, "lib")
    cuda = os.path.join(os.path.dirname(os.path.dirname(os.path.realpath(_nvcc()))), "include")
    cmd = [host_cxx, "-O2", "-std=c++17", "-fPIC", "-shared", "-I" + include, "-I" + os.path.join(include, "torch", "csrc", "api", "include"),
           "-I" + sysconfig.get_paths()["include"], "-I" + cuda, os.path.join(CSRC, "tensor_calls.cpp"), "-o", TENSOR_CALLS, "-L" + HERE,
           "-l:" + os.path.basename(LIB), "-Wl,-rpath,$ORIGIN", "-L" + lib, "-lc10", "-lc10_cuda", "-ltorch", "-ltorch_cpu", "-ltorch_cuda", "-ltorch_python",
           "-Wl,-rpath," + lib]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if verbose or res.returncode:
        sys.stderr.write(res.stdout + res.stderr)
    if res.returncode:
        sys.stderr.write(f"building bullet_b200._tensor_calls for {_made_for()} failed: bullet_b200.ops is not built\n")
        return None
    with open(MADE_FOR, "w") as f:
        f.write(_made_for())
    return TENSOR_CALLS


if __name__ == "__main__":
    print(build(force=True, verbose="--verbose" in sys.argv))
