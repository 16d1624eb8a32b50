"""Builds the in-tree shared library `csrc/libadhip.so` with hipcc for gfx950.

The library holds the host side of the device (IR parser, lowering, code generator, runtime), whose device code is
generated per program and compiled for gfx950 by hipRTC, and the operators on device arrays (`csrc/*.hip`), whose kernels
are compiled here."""
from __future__ import annotations

import glob
import os
import subprocess
import tempfile
from concurrent.futures import ThreadPoolExecutor

_PKG_DIR = os.path.dirname(os.path.abspath(__file__))
# Matrix instructions add up in the registers that vector instructions reach too: by default a kernel that has all of a SIMD's
# registers carries its sums to the other half and back in every step.
KERNEL_FLAGS = ["-O3", "-mllvm", "-amdgpu-mfma-vgpr-form"]
# Sums that fill one half are better off in the other.
WIDE_SUMS = {"operator_attention_backward_f32_wide.hip"}
CSRC = os.path.join(os.path.dirname(_PKG_DIR), "csrc")


def build_library(verbose: bool = False) -> str:
    hipcc = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
    out = os.path.join(CSRC, "libadhip.so")
    flags = ["--offload-arch=gfx950", "-std=c++17", "-fPIC", "-Wall", "-Wno-unused-function", "-Xclang", "-target-feature", "-Xclang",
             "-packed-fp32-ops"]
    with tempfile.TemporaryDirectory() as work:
        steps, objects = [], []
        # kernels first: their files take longest
        for src in sorted(glob.glob(os.path.join(CSRC, "*.hip"))) + sorted(glob.glob(os.path.join(CSRC, "*.cpp"))):
            objects.append(os.path.join(work, os.path.basename(src) + ".o"))
            steps.append([hipcc, *flags, *(["-O2"] if src.endswith(".cpp") else ["-O3"] if os.path.basename(src) in WIDE_SUMS else KERNEL_FLAGS), "-c", src, "-o", objects[-1]])
        steps_at_once = int(os.environ.get("MAX_JOBS", min(16, os.cpu_count() or 1)))
        with ThreadPoolExecutor(max(1, steps_at_once)) as pool:
            def compile_one(cmd):
                if verbose:
                    print(" ".join(cmd))
                done = subprocess.run(cmd, capture_output=True, text=True)
                # hipcc's host pass does not know the device feature that is switched off
                said = [x for x in done.stderr.splitlines() if "is not a recognized feature for this target" not in x]
                if said:
                    print("\n".join(said))
                if done.returncode != 0:
                    raise RuntimeError(f"hipcc failed on {cmd[-3]}")
            list(pool.map(compile_one, steps))
        link = [hipcc, "--offload-arch=gfx950", "-fPIC", "-shared", "-o", out, *objects, "-lhiprtc"]
        if verbose:
            print(" ".join(link))
        subprocess.check_call(link)
    return out


def build_cxx_smoke(verbose: bool = False) -> str:
    """Compile tests/cxx/cabi_smoke.cpp (plain C++ against include/adhip.h) and link it with the library."""
    root = os.path.dirname(os.path.dirname(_PKG_DIR))
    src = os.path.join(root, "tests", "cxx", "cabi_smoke.cpp")
    out = os.path.join(root, "tests", "cxx", "cabi_smoke")
    cmd = ["g++", "-O2", "-std=c++17", "-Wall", "-o", out, src, "-L" + CSRC, "-ladhip", "-Wl,-rpath," + CSRC,
           "-Wl,-rpath,/opt/rocm/lib"]
    if verbose:
        print(" ".join(cmd))
    subprocess.check_call(cmd)
    return out


def build_overlap_probe(verbose: bool = False) -> str:
    """Compile tests/cxx/mfma_valu_overlap.cpp (a hardware premise of the matrix kernels, measured) for gfx950."""
    root = os.path.dirname(os.path.dirname(_PKG_DIR))
    src = os.path.join(root, "tests", "cxx", "mfma_valu_overlap.cpp")
    out = os.path.join(root, "tests", "cxx", "mfma_valu_overlap")
    hipcc = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
    cmd = [hipcc, "--offload-arch=gfx950", "-O3", "-std=c++17", "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
           "-o", out, src]
    if verbose:
        print(" ".join(cmd))
    subprocess.check_call(cmd)
    return out


if __name__ == "__main__":
    print(build_library(verbose=True))
