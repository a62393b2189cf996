"""Build recipe for the native code, output in-tree: the library (one nvcc call, sm_100a only) and the PyTorch binding of the feed-forward
products (one C++ file against PyTorch's headers, no kernel in it)."""
import os
import shutil
import subprocess
import sys
import sysconfig

PKG = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(PKG, "csrc")
LIB = os.path.join(PKG, "libproteus_b200.so")
HEADER = os.path.join(os.path.dirname(PKG), "include", "proteus_b200.h")
TORCH_OPS = os.path.join(CSRC, "torch_ops.cpp")
TORCH_OPS_LIB = os.path.join(PKG, "_torch_ops.so")

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17",
    "-shared", "-Xcompiler", "-fPIC",
]


def sources():
    return sorted(os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".cu", ".cuh"))) + [HEADER]


def _older(target, inputs):
    return not os.path.exists(target) or any(os.path.getmtime(s) > os.path.getmtime(target) for s in inputs)


def is_stale():
    return _older(LIB, sources())


def _run(cmd):
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"{os.path.basename(cmd[0])} failed:\n" + res.stdout + res.stderr)
    return res


def build(force=False, verbose=False):
    """Compile csrc/api.cu (which includes every kernel) into libproteus_b200.so, and csrc/torch_ops.cpp into _torch_ops.so."""
    if force or _older(TORCH_OPS_LIB, [TORCH_OPS, HEADER]):
        build_torch_ops()
    if not force and not is_stale():
        return LIB
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    res = _run([nvcc] + NVCC_FLAGS + (["-Xptxas", "-v"] if verbose else []) + ["-o", LIB, os.path.join(CSRC, "api.cu")])
    if verbose:
        print(res.stderr)
    return LIB


def build_torch_ops():
    import torch
    from torch.utils import cpp_extension
    dirs = cpp_extension.include_paths(device_type="cuda") + [sysconfig.get_paths()["include"]]
    libs = os.path.join(os.path.dirname(torch.__file__), "lib")
    _run([shutil.which("g++") or "c++", "-O2", "-std=c++17", "-shared", "-fPIC", "-fvisibility=hidden", "-DTORCH_EXTENSION_NAME=_torch_ops",
          f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}"] + [f for d in dirs for f in ("-isystem", d)] +
         [TORCH_OPS, "-o", TORCH_OPS_LIB, f"-L{libs}", f"-Wl,-rpath,{libs}", "-ltorch", "-ltorch_cpu", "-ltorch_cuda", "-ltorch_python", "-lc10",
          "-lc10_cuda"])
    return TORCH_OPS_LIB


if __name__ == "__main__":
    print(build(force=True, verbose="-v" in sys.argv))
