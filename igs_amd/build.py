"""Builds igs_amd/libigs_hip.so (the C-ABI shared library) with hipcc for gfx950, and igs_amd/_igs_torch.so
(host code: the feature operators' autograd nodes around that library) with g++ against the installed torch.

Usage: python -m igs_amd.build            (from the repository root)
hipcc cross-compiles without a GPU; the built library sits in-tree next to this file.
"""
from __future__ import annotations

import os
import subprocess
import sys
import tempfile

PKG = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG)
SOURCES = [os.path.join(PKG, "csrc", f) for f in ("igs_gs2d.hip", "igs_feature.hip", "igs_norm.hip")]
LIB = os.path.join(PKG, "libigs_hip.so")
TORCH_SOURCE = os.path.join(PKG, "csrc", "igs_torch.cpp")
TORCH_LIB = os.path.join(PKG, "_igs_torch.so")

# Packed-fp32 instruction selection is switched off for all device code.
HIPCC_FLAGS = [
    "-O3",
    "-std=c++17",
    "--offload-arch=gfx950",
    "-fPIC",
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    # matrix-core results land in ordinary VGPRs (the vector ALU reads them without a copy out of
    # the accumulation registers); only the diversity-loss kernel uses the matrix cores
    "-mllvm", "-amdgpu-mfma-vgpr-form=1",
    "-I", os.path.join(ROOT, "include"),
]


def build(verbose: bool = True, extra=()) -> str:
    """Every unit by a compiler of its own, side by side, then the library."""
    hipcc = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
    with tempfile.TemporaryDirectory() as tmp:
        objects = [os.path.join(tmp, os.path.basename(s) + ".o") for s in SOURCES]
        cmds = [[hipcc, *HIPCC_FLAGS, *extra, "-c", s, "-o", o] for s, o in zip(SOURCES, objects)] + [torch_command()]
        running = []
        for cmd in cmds:
            if verbose:
                print(" ".join(cmd), flush=True)
            running.append(subprocess.Popen(cmd))
        for p in [p for p in running if p.wait()]:
            raise subprocess.CalledProcessError(p.returncode, p.args)
        link = [hipcc, "--offload-arch=gfx950", "-fPIC", "-shared", "-o", LIB, *objects]
        if verbose:
            print(" ".join(link), flush=True)
        subprocess.check_call(link)
    return LIB


def torch_command():
    import sysconfig

    import torch
    from torch.utils import cpp_extension

    lib = os.path.join(os.path.dirname(torch.__file__), "lib")
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden", "-DNDEBUG",
           "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}",
           "-DTORCH_EXTENSION_NAME=_igs_torch", "-I", os.path.join(ROOT, "include")]
    for path in [*cpp_extension.include_paths(), os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "include"),
                 sysconfig.get_paths()["include"]]:
        cmd += ["-isystem", path]
    cmd += [TORCH_SOURCE, "-o", TORCH_LIB, "-L", lib, "-ltorch", "-ltorch_cpu", "-ltorch_python", "-lc10", "-lc10_hip", "-ldl"]
    return cmd


def is_stale() -> bool:
    if not os.path.exists(LIB) or not os.path.exists(TORCH_LIB):
        return True
    t = min(os.path.getmtime(LIB), os.path.getmtime(TORCH_LIB))
    csrc = os.path.join(PKG, "csrc")
    deps = [os.path.join(csrc, f) for f in os.listdir(csrc)] + [os.path.join(ROOT, "include", "igs_hip.h")]
    return any(os.path.getmtime(d) > t for d in deps)


if __name__ == "__main__":
    build(extra=sys.argv[1:])
