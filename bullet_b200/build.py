"""Builds libbullet_b200.so in-tree with nvcc for sm_100a (cross-compiles without a GPU), and the module of the tensor calls (ops.py).

    python -m bullet_b200.build [--verbose]
"""
from __future__ import annotations

import importlib.util
import os
import shutil
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libbullet_b200.so")
TENSOR_CALLS = os.path.join(HERE, "_tensor_calls.so")
SOURCES = ["net.cu", "op_ft_forward.cu", "op_rows.cu", "op_dense.cu", "gave_up.cu", "probe.cu", "host_pack.cpp", "checkpoint.cpp", "saved_format.cpp"]


def _nvcc() -> str:
    for cand in (shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found: bullet_b200 has no CPU fallback and cannot be built without the CUDA toolkit")


def _torch_dir() -> str | None:
    spec = importlib.util.find_spec("torch")
    return os.path.dirname(spec.origin) if spec else None


def _stale() -> bool:
    outputs = [LIB] + ([TENSOR_CALLS] if _torch_dir() else [])
    if not all(os.path.exists(p) for p in outputs):
        return True
    built = min(os.path.getmtime(p) for p in outputs)
    deps = [os.path.join(CSRC, f) for f in os.listdir(CSRC)] + [os.path.join(HERE, "..", "include", "bullet_b200.h")]
    return any(os.path.getmtime(p) > built for p in deps)


def build(force: bool = False, verbose: bool = False) -> str:
    if not force and not _stale():
        return LIB
    host_cxx = "/usr/bin/g++" if os.path.exists("/usr/bin/g++") else "g++"  # needs libgomp
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
    build_tensor_calls(host_cxx, verbose)
    return LIB


def build_tensor_calls(host_cxx: str, verbose: bool = False) -> str | None:
    """The module behind ops.py, against the torch that is installed; None without one (the library needs none)."""
    torch_dir = _torch_dir()
    if torch_dir is None:
        sys.stderr.write("torch is not installed: bullet_b200.ops is not built\n")
        return None
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
        raise RuntimeError("building bullet_b200._tensor_calls failed")
    return TENSOR_CALLS


if __name__ == "__main__":
    print(build(force=True, verbose="--verbose" in sys.argv))
