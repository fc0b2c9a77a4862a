"""Ahead-of-time build of the HIP library for gfx950 (MI355X) and of the host extension module.

The reference compiles its kernels at run time with NVRTC after text substitution
(models/cuda_funcs/kernel_manager.py:116-167); here every supported constant set is a template
instantiation compiled once by hipcc into ``libcrystalframer_hip.so`` next to this file.
"""
from __future__ import annotations

import concurrent.futures
import os
import shutil
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB_NAME = "libcrystalframer_hip.so"
LIB_PATH = os.path.join(HERE, LIB_NAME)
HOST_PATH = os.path.join(HERE, "_host.so")

LIB_SOURCES = ("crystalframer_hip", "training_ops", "residual_norm_f32", "residual_norm_bf16", "residual_norm_f16",
               "sequence_attention_ops", "sequence_attention_f32", "sequence_attention_bf16", "sequence_attention_f16")

HIPCC_FLAGS = [
    "-O3", "--offload-arch=gfx950", "-std=c++17", "-fPIC",
    # packed FP32 instructions are kept out of the generated code
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
]

# results of matrix instructions stay in the registers that all others use: sums that are scaled between products are not moved
SOURCE_FLAGS = {name: ["-mllvm", "-amdgpu-mfma-vgpr-form=1"] for name in LIB_SOURCES if name.startswith("sequence_attention_")}


def hipcc_path() -> str:
    for cand in (shutil.which("hipcc"), "/opt/rocm/bin/hipcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("hipcc not found (looked on PATH and in /opt/rocm/bin)")


def _run(cmd, verbose):
    if verbose:
        print("[crystalframer_amd] " + " ".join(cmd), flush=True)
    return subprocess.run(cmd, capture_output=True, text=True)


def build_library(verbose: bool = True) -> str:
    """Compile the sources of csrc -> libcrystalframer_hip.so (always recompiles), side by side, and link them."""
    # CFH_EXTRA_HIPCC_FLAGS: extra flags for diagnostics builds (e.g. -DCFH_PHASE_TIMING)
    extra = os.environ.get("CFH_EXTRA_HIPCC_FLAGS", "").split()
    tmp = LIB_PATH + ".tmp"
    objects = [os.path.join(HERE, name + ".o") for name in LIB_SOURCES]
    cmds = [[hipcc_path(), *HIPCC_FLAGS, *SOURCE_FLAGS.get(name, []), *extra, "-c", "-o", obj, os.path.join(CSRC, name + ".hip")]
            for name, obj in zip(LIB_SOURCES, objects)]
    try:
        with concurrent.futures.ThreadPoolExecutor(len(cmds)) as pool:
            failed = [res for res in pool.map(lambda cmd: _run(cmd, verbose), cmds) if res.returncode != 0]
        if not failed:
            res = _run([hipcc_path(), "--offload-arch=gfx950", "-shared", "-fPIC", "-o", tmp, *objects], verbose)
            failed = [res] if res.returncode != 0 else []
    finally:
        for obj in objects:
            if os.path.exists(obj):
                os.remove(obj)
    if failed:
        sys.stderr.write("".join(res.stdout + res.stderr for res in failed))
        raise RuntimeError("hipcc failed building " + LIB_NAME)
    os.replace(tmp, LIB_PATH)
    return LIB_PATH


def build_host(verbose: bool = True) -> str:
    """Compile csrc/host_module.cpp -> _host.so, the Python extension module around the whole-model pass (always recompiles).
    Host code only: the framework's headers and libraries, no kernels."""
    import torch
    from torch.utils import cpp_extension
    tmp = HOST_PATH + ".tmp"
    inc = [*cpp_extension.include_paths(), sysconfig.get_paths()["include"], "/opt/rocm/include"]
    libs = os.path.join(os.path.dirname(torch.__file__), "lib")
    cmd = [shutil.which("g++") or "g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", *("-I" + p for p in inc), "-o", tmp,
           os.path.join(CSRC, "host_module.cpp"), "-L" + libs, "-lc10", "-lc10_hip", "-ltorch_cpu", "-ltorch", "-ltorch_python"]
    if verbose:
        print("[crystalframer_amd] " + " ".join(cmd), flush=True)
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        sys.stderr.write(res.stdout + res.stderr)
        raise RuntimeError("g++ failed building _host.so")
    os.replace(tmp, HOST_PATH)
    return HOST_PATH


if __name__ == "__main__":
    print(build_library())
    print(build_host())
