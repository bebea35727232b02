"""Build the gfx950 HIP extension IN-TREE.

The built .so lands in runbookai_amd/ops/_build/, so that it goes where a copy
of the tree goes (a JIT cache under ~/.cache would not). hipcc cross-compiles
for gfx950 without a GPU present.
"""
from __future__ import annotations

import os
import sys

OPS_DIR = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(OPS_DIR, "csrc")
BUILD_DIR = os.path.join(OPS_DIR, "_build")
EXT_NAME = "runbookai_hip_ops"

SOURCES = [
    os.path.join(CSRC, "bindings.cpp"),
    os.path.join(CSRC, "norm_elem.hip"),
    os.path.join(CSRC, "attention.hip"),
    os.path.join(CSRC, "flash_prefill.hip"),
    os.path.join(CSRC, "flash_prefill2.hip"),
    os.path.join(CSRC, "skinny_gemm.hip"),
    os.path.join(CSRC, "decode_gemv.hip"),
    os.path.join(CSRC, "retrieval_sampling.hip"),
    os.path.join(CSRC, "training.cpp"),
    os.path.join(CSRC, "packed_attn.hip"),
    os.path.join(CSRC, "cross_entropy.hip"),
    os.path.join(CSRC, "grad_norm.hip"),
]

# hipcc would otherwise form packed fp32 instructions from ordinary float code,
# some of which have given wrong results on this hardware. (The host pass does
# not know the feature and says so.)
HIP_FLAGS = ["-O3", "-std=c++17",
             "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]


def build(verbose: bool = False):
    """Compile the extension; returns the imported module.

    Everything is compiled, whatever an earlier build left: the build tool does
    not know which headers a kernel includes, so a kernel whose argument struct
    changed in a header would keep its old object and read the new struct by the
    old one's layout."""
    os.environ.setdefault("PYTORCH_ROCM_ARCH", "gfx950")
    os.makedirs(BUILD_DIR, exist_ok=True)
    for fn in os.listdir(BUILD_DIR):
        if fn.endswith((".o", ".so")):
            os.remove(os.path.join(BUILD_DIR, fn))
    from torch.utils.cpp_extension import load

    module = load(
        name=EXT_NAME,
        sources=SOURCES,
        build_directory=BUILD_DIR,
        extra_cflags=["-O3"],
        extra_cuda_cflags=HIP_FLAGS,
        verbose=verbose,
        with_cuda=True,  # ROCm build: drives hipcc for the .hip sources
    )
    return module


def load_prebuilt():
    """Import a previously-built .so without invoking the compiler."""
    import importlib.util

    for fn in os.listdir(BUILD_DIR) if os.path.isdir(BUILD_DIR) else []:
        if fn.startswith(EXT_NAME) and fn.endswith(".so"):
            spec = importlib.util.spec_from_file_location(EXT_NAME,
                                                          os.path.join(BUILD_DIR, fn))
            mod = importlib.util.module_from_spec(spec)
            spec.loader.exec_module(mod)
            return mod
    return None


if __name__ == "__main__":
    build(verbose=True)
    print("built", EXT_NAME, "->", BUILD_DIR)
