"""Builds libssla_b200.so in-tree (nvcc, sm_100a).

The library is a plain C-ABI shared object (include/ssla_b200.h); the CUDA
runtime is linked statically so the .so needs only the driver on the GPU box.
Flags: -fmad=false keeps every floating-point contraction explicit (the
kernels write fmaf where the reference's arithmetic is a fused
multiply-add), which is what makes results bit-identical to the CPU oracle.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
REPO = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libssla_b200.so")
# The same library under the reference's name, for callers that load the
# s01g_* ABI as libstage01_to_gpu.so (orin/orin/hybrid_common.py S01gAPI).
S01G_LIB = os.path.join(HERE, "libstage01_to_gpu.so")
SOURCES = ["ssla_kernels.cu", "ssla_engine.cu", "ssla_weights.cpp", "ssla_noalloc.cu", "ssla_s01g.cpp", "ssla_step.cu", "ssla_live.cu", "ssla_dump.cpp", "ssla_strip.cu", "ssla_rings.cu", "ssla_replay.cpp", "ssla_head_tc.cu", "ssla_linattn.cu", "ssla_linattn_chunk.cu", "ssla_statecache.cu", "ssla_groupnorm.cu"]
HEADERS = ["ssla_device.cuh", "ssla_kernels.cuh", "ssla_weights.h", "ssla_cluster.cuh", "ssla_ops.cuh", "ssla_linattn.cuh", "ssla_linattn_tc.cuh"]
NVCC_FLAGS = ["-O3", "-std=c++17", "-gencode", "arch=compute_100a,code=sm_100a",
              "-lineinfo", "-fmad=false", "-Xcompiler", "-fPIC", "-shared",
              "-cudart", "static"]


def _nvcc() -> str:
    for c in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", "nvcc"):
        if c and (os.path.isabs(c) and os.path.exists(c) or not os.path.isabs(c)):
            return c
    return "nvcc"


def _stale() -> bool:
    if not os.path.exists(LIB):
        return True
    t = os.path.getmtime(LIB)
    deps = [os.path.join(CSRC, f) for f in SOURCES + HEADERS]
    deps += [os.path.join(REPO, "include", f) for f in ("ssla_b200.h", "ssla_abi_types.h", "stage01_to_gpu.h", "ssla_ops.h")]
    return any(os.path.getmtime(d) > t for d in deps) or not os.path.exists(S01G_LIB)


# The stage-2/3 ring consumer module (kernels/), prebuilt for sm_100a: the
# same source the reference's runners NVRTC-compile, loadable by name.
KERNELS = os.path.join(HERE, "kernels")
CONSUMER_SRC = os.path.join(KERNELS, "ssla_s2_s3_head_celled.cuh")
CONSUMER_HDR = os.path.join(KERNELS, "proto_layer_pair.cuh")
CONSUMER_CUBIN = os.path.join(HERE, "ssla_s2s3_consumer.cubin")


def build_consumer(force: bool = False, verbose: bool = False) -> str:
    if (not force and os.path.exists(CONSUMER_CUBIN) and
            os.path.getmtime(CONSUMER_CUBIN) >= max(os.path.getmtime(CONSUMER_SRC), os.path.getmtime(CONSUMER_HDR))):
        return CONSUMER_CUBIN
    cmd = [_nvcc(), "-x", "cu", "-cubin", "-O3", "-std=c++17", "-gencode", "arch=compute_100a,code=sm_100a",
           "-lineinfo", f"-I{KERNELS}", CONSUMER_SRC, "-o", CONSUMER_CUBIN]
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.run(cmd, check=True)
    return CONSUMER_CUBIN


# The repeated calls of ops.py in one step: a Python extension module over
# torch's tensors (the library itself stays free of torch).  It fits the torch
# and Python that it was built with; the stamp beside it names them.
OPS_TORCH_SRC = os.path.join(CSRC, "ssla_ops_torch.cpp")
OPS_TORCH = os.path.join(HERE, "_ops_torch.so")
OPS_TORCH_STAMP = os.path.join(HERE, "_build", "ops_torch.stamp")


def ops_torch_abi() -> str:
    import sysconfig

    import torch
    return f"torch {torch.__version__} python {sysconfig.get_config_var('SOABI')}"


def _read(path: str) -> str:
    try:
        with open(path) as f:
            return f.read()
    except OSError:
        return ""


def build_ops_torch(force: bool = False, verbose: bool = False) -> str:
    abi = ops_torch_abi()
    deps = [OPS_TORCH_SRC] + [os.path.join(REPO, "include", f) for f in ("ssla_b200.h", "ssla_ops.h")]
    if (not force and os.path.exists(OPS_TORCH) and os.path.getmtime(OPS_TORCH) >= max(map(os.path.getmtime, deps)) and
            _read(OPS_TORCH_STAMP) == abi):
        return OPS_TORCH
    import sysconfig

    import torch
    from torch.utils import cpp_extension
    dirs = [os.path.join(REPO, "include"), sysconfig.get_paths()["include"], "/usr/local/cuda/include",
            *cpp_extension.include_paths()]
    lib = os.path.join(os.path.dirname(torch.__file__), "lib")
    cmd = ["g++", "-O2", "-std=c++17", "-shared", "-fPIC", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           *[f"-I{d}" for d in dirs], OPS_TORCH_SRC, "-o", OPS_TORCH, f"-L{lib}", "-lc10", "-lc10_cuda", "-ltorch_cpu",
           "-ltorch_python"]
    if verbose:
        print(" ".join(cmd), flush=True)
    # a module of another torch would take the process down when it is imported: it goes first
    if os.path.exists(OPS_TORCH):
        os.remove(OPS_TORCH)
    subprocess.run(cmd, check=True)
    os.makedirs(os.path.dirname(OPS_TORCH_STAMP), exist_ok=True)
    with open(OPS_TORCH_STAMP, "w") as f:
        f.write(abi)
    return OPS_TORCH


def build(force: bool = False, verbose: bool = False) -> str:
    """The library and the consumer module; then the extension module, which
    may fail (no torch, or one without CUDA): ops.py does without it."""
    build_consumer(force=force, verbose=verbose)
    lib = build_library(force=force, verbose=verbose)
    try:
        build_ops_torch(force=force, verbose=verbose)
    except (ImportError, OSError, subprocess.CalledProcessError) as e:
        print(f"ssla_rt_b200: repeated operator calls go without their extension module: {e}", file=sys.stderr)
    return lib


def build_library(force: bool = False, verbose: bool = False) -> str:
    if not force and not _stale():
        return LIB
    cmd = [_nvcc(), *NVCC_FLAGS, f"-I{os.path.join(REPO, 'include')}", f"-I{CSRC}",
           *[os.path.join(CSRC, f) for f in SOURCES], "-o", LIB]
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.run(cmd, check=True)
    shutil.copyfile(LIB, S01G_LIB)
    os.chmod(S01G_LIB, 0o755)
    return LIB


if __name__ == "__main__":
    build(force="--force" in sys.argv, verbose=True)
    print(LIB)
