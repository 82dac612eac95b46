"""Ahead-of-time build of libb200moe.so (sm_100a only) with nvcc; no JIT cache, the library stays in-tree.

    python -m kernelschema_b200.build [--force] [--verbose]
"""
from __future__ import annotations

import os
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libb200moe.so")
SHIM = os.path.join(HERE, "_b200moe_shim.so")
TORCH_CALLS = os.path.join(HERE, "_b200moe_torch.so")
TORCH_STAMP = os.path.join(HERE, "build", "torch_calls.torch")      # the torch and Python that TORCH_CALLS was built for
SOURCES = ["quantize.cu", "router.cu", "route_map.cu", "gather.cu", "finalize.cu", "gemm_nvfp4.cu", "gemm_w4a16.cu", "gemm_w4a16_decode.cu", "gemm_w4a16_expand.cu", "ep_exchange.cu", "rowquant.cu", "gemm_8bit.cu", "gemm_8bit_decode.cu", "route_order.cu", "api.cu"]
HEADERS = ["gemm_8bit.cuh", "gemm_8bit_clusters.cuh", "gemm_8bit_plan.cuh", "kernels.cuh", "ptx.cuh", "quantize.cuh", "rows.cuh", "topk.cuh", "w4a16.cuh", os.path.join("..", "..", "include", "b200moe.h")]
NVCC_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17", "-Xcompiler", "-fPIC",
              "-Xptxas", "-v"]


def _nvcc() -> str:
    for cand in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", "nvcc"):
        if cand and (os.path.sep not in cand or os.path.exists(cand)):
            return cand
    raise RuntimeError("nvcc not found")


def _stale(target: str, deps: list[str]) -> bool:
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


def build(force: bool = False, verbose: bool = False) -> str:
    """Compile every CUDA source for sm_100a and link the shared library. Returns its path."""
    nvcc = _nvcc()
    objdir = os.path.join(HERE, "build")
    os.makedirs(objdir, exist_ok=True)
    headers = [os.path.join(CSRC, h) for h in HEADERS]

    def compile_one(src: str) -> str:
        obj = os.path.join(objdir, src.replace(".cu", ".o"))
        path = os.path.join(CSRC, src)
        if force or _stale(obj, [path] + headers):
            cmd = [nvcc, *NVCC_FLAGS, "-c", path, "-o", obj]
            res = subprocess.run(cmd, capture_output=True, text=True)
            with open(obj + ".log", "w") as f:
                f.write(" ".join(cmd) + "\n" + res.stdout + res.stderr)
            if res.returncode != 0:
                raise RuntimeError(f"nvcc failed on {src}:\n{res.stderr}")
            if verbose:
                print(res.stderr)
        return obj

    with ThreadPoolExecutor(max_workers=min(8, len(SOURCES))) as ex:
        objs = list(ex.map(compile_one, SOURCES))
    if force or _stale(LIB, objs):
        cmd = [nvcc, "-shared", "-o", LIB, *objs, "-gencode", "arch=compute_100a,code=sm_100a"]
        res = subprocess.run(cmd, capture_output=True, text=True)
        if res.returncode != 0:
            raise RuntimeError("link failed:\n" + res.stderr)
    build_shim(force)
    build_torch_calls(force)
    return LIB


def build_shim(force: bool = False) -> str:
    """Compile the pybind11 shim (plain C++, links against the in-tree libb200moe.so through $ORIGIN)."""
    import sysconfig
    import pybind11
    src = os.path.join(CSRC, "shim.cpp")
    if force or _stale(SHIM, [src, LIB, os.path.join(CSRC, "..", "..", "include", "b200moe.h")]):
        cmd = ["g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-fvisibility=hidden", "-I", pybind11.get_include(), "-I",
               sysconfig.get_paths()["include"], src, "-o", SHIM, "-L", HERE, "-lb200moe", "-Wl,-rpath,$ORIGIN"]
        res = subprocess.run(cmd, capture_output=True, text=True)
        if res.returncode != 0:
            raise RuntimeError("shim build failed:\n" + res.stderr)
    return SHIM


def build_torch_calls(force: bool = False) -> str:
    """Compile the calls on torch tensors (C++ against torch's headers; links the in-tree libb200moe.so through $ORIGIN), again where torch or
    Python is another than it was built for."""
    import torch
    src = os.path.join(CSRC, "torch_calls.cpp")
    wanted = f"torch {torch.__version__} python {sys.version_info[0]}.{sys.version_info[1]}\n"
    built_for = None
    if os.path.exists(TORCH_STAMP):
        with open(TORCH_STAMP) as f:
            built_for = f.read()
    if force or built_for != wanted or _stale(TORCH_CALLS, [src, LIB, os.path.join(CSRC, "..", "..", "include", "b200moe.h")]):
        import sysconfig
        base = os.path.dirname(torch.__file__)
        cuda = os.path.dirname(os.path.dirname(_nvcc()))
        cmd = ["g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-fvisibility=hidden", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}",
               "-I", os.path.join(base, "include"), "-I", os.path.join(base, "include", "torch", "csrc", "api", "include"), "-I",
               os.path.join(cuda, "include"), "-I", sysconfig.get_paths()["include"], src, "-o", TORCH_CALLS, "-L", HERE, "-lb200moe", "-L",
               os.path.join(base, "lib"), "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_cuda", "-ltorch_python", "-Wl,-rpath,$ORIGIN"]
        res = subprocess.run(cmd, capture_output=True, text=True)
        if res.returncode != 0:
            raise RuntimeError("build of the torch calls failed:\n" + res.stderr)
        os.makedirs(os.path.dirname(TORCH_STAMP), exist_ok=True)
        with open(TORCH_STAMP, "w") as f:
            f.write(wanted)
    return TORCH_CALLS


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="--verbose" in sys.argv))
