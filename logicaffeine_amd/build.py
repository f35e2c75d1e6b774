"""Build recipe of liblgx (no cmake, no JIT cache: everything lands in-tree).

    lgx_kernels.hsaco  hipcc --offload-arch=gfx950 (device code only) per kernel file, linked
    liblgx.so          g++ host launcher over the HIP module API

Run as ``python -m logicaffeine_amd.build``; ``__graft_entry__.build()`` calls
:func:`build`.  Both artefacts sit next to this file, which is where
``lgx_ctx_create(dev, NULL, ...)`` looks for the code object.
"""
from __future__ import annotations

import concurrent.futures
import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
ROCM = os.environ.get("ROCM_PATH", "/opt/rocm")
ARCH = "gfx950"

HSACO = os.path.join(HERE, "lgx_kernels.hsaco")
LIB = os.path.join(HERE, "liblgx.so")

# -ffp-contract=off: no implicit fusion, the float schedule is what the source
# says.  Correctly rounded binary32 division and square root.  Packed-FP32
# instructions disabled (v_pk_*_f32 are never generated).  MFMA destinations
# in VGPRs.
HIP_FLAGS = [
    "--offload-device-only", "--no-gpu-bundle-output", f"--offload-arch={ARCH}", "-O3", "-std=c++17",
    "-ffp-contract=off", "-fhip-fp32-correctly-rounded-divide-sqrt",
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    # MFMA results in ordinary VGPRs (gfx950 allows it): the epilogues read
    # them directly instead of copying each value out of an AGPR first
    "-mllvm", "-amdgpu-mfma-vgpr-form",
]


def _run(cmd):
    print("[lgx build]", " ".join(cmd), flush=True)
    subprocess.run(cmd, check=True)


KERNEL_SOURCES = ["lgx_kernels.hip", "lgx_pages.hip", "lgx_tree.hip", "lgx_tree_attn.hip", "lgx_filter.hip"]
BUILD_DIR = os.path.join(HERE, "_build")


def _compile_kernels(source: str) -> str:
    """One kernel file to an AMDGPU object, by way of its assembly (hipcc itself
    links whatever it compiles for the device)."""
    stem = os.path.join(BUILD_DIR, os.path.splitext(source)[0])
    _run([os.path.join(ROCM, "bin", "hipcc"), *HIP_FLAGS, "-S", "-I", CSRC, "-o", stem + ".s", os.path.join(CSRC, source)])
    with open(stem + ".s", "a") as f:
        # up to the next file's first kernel (256-byte aligned) with s_nop, not with zeros
        f.write("\n\t.text\n\t.p2alignl 8, 0xbf800000\n")
    _run([os.path.join(ROCM, "llvm", "bin", "clang"), "--target=amdgcn-amd-amdhsa", f"-mcpu={ARCH}", "-c", "-o", stem + ".o",
          stem + ".s"])
    os.remove(stem + ".s")
    return stem + ".o"


def build_kernels() -> str:
    """The code object of all kernel files, compiled side by side."""
    os.makedirs(BUILD_DIR, exist_ok=True)
    with concurrent.futures.ThreadPoolExecutor(len(KERNEL_SOURCES)) as pool:
        objects = list(pool.map(_compile_kernels, KERNEL_SOURCES))
    tmp = HSACO + ".tmp"
    _run([os.path.join(ROCM, "llvm", "bin", "ld.lld"), "-shared", "--no-undefined", "-o", tmp, *objects])
    os.replace(tmp, HSACO)
    return HSACO


HOST_SOURCES = ["lgx_host.cpp", "lgx_glue.cpp", "lgx_model.cpp", "lgx_gen.cpp", "lgx_gguf.cpp",
                "lgx_f16gemm.cpp", "lgx_kv8.cpp", "lgx_pages.cpp",
                "lgx_tree.cpp"]


def build_scratch() -> str:
    """lgx_scratch.hip: host code plus a gfx950 code object holding only the
    no-alloc entry point's device scratch array, registered with the HIP
    runtime when liblgx.so loads."""
    os.makedirs(BUILD_DIR, exist_ok=True)
    obj = os.path.join(BUILD_DIR, "lgx_scratch.o")
    _run([os.path.join(ROCM, "bin", "hipcc"), "-c", "-fPIC", "-O2", "-std=c++17", f"--offload-arch={ARCH}",
          "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
          "-I", CSRC, "-o", obj, os.path.join(CSRC, "lgx_scratch.hip")])
    return obj


def build_host() -> str:
    srcs = [os.path.join(CSRC, s) for s in HOST_SOURCES]
    scratch_obj = build_scratch()
    tmp = LIB + ".tmp"
    _run(["g++", "-O2", "-fPIC", "-shared", "-std=c++17", "-ffp-contract=off", "-Wall", "-Wextra", "-pthread",
          "-D__HIP_PLATFORM_AMD__", f"-I{ROCM}/include", "-I", CSRC,
          "-o", tmp, *srcs, scratch_obj, f"-L{ROCM}/lib", "-lamdhip64", "-lhipblaslt", f"-Wl,-rpath,{ROCM}/lib", "-ldl"])
    os.replace(tmp, LIB)
    return LIB


def build() -> None:
    build_kernels()
    build_host()


if __name__ == "__main__":
    build()
    sys.exit(0)
