"""Builds libnrq.so (gfx950 only) from nightrun_amd/csrc/*.hip, and _serve.so,
the Python side of the serving operators over torch tensors, from csrc/serve_bind.cpp.

    python -m nightrun_amd.build

Each source is compiled to an object under nightrun_amd/_build/ in parallel,
then linked into nightrun_amd/libnrq.so next to this file. hipcc
cross-compiles for gfx950 without a GPU present.
"""
from __future__ import annotations

import concurrent.futures as cf
import glob
import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
BUILD = os.path.join(HERE, "_build")
LIB = os.path.join(HERE, "libnrq.so")
BIND = os.path.join(HERE, "_serve.so")
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")

# -ffp-contract=off: a*b+c stays two rounded operations, as in the Rust
# reference (which never contracts); fmaf() marks the reference's FMAs.
# -packed-fp32-ops: no v_pk_*_f32 instructions in generated code.
HIP_FLAGS = [
    "--offload-arch=gfx950",
    "-O3",
    "-std=c++17",
    "-fPIC",
    "-ffp-contract=off",
    "-fno-gpu-rdc",
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    # MFMA results in VGPRs (gfx950 allows it): no v_accvgpr_read per result
    "-mllvm", "-amdgpu-mfma-vgpr-form",
    "-Wall",
    "-Wno-unused-function",
]


def _compile(src: str) -> str:
    obj = os.path.join(BUILD, os.path.basename(src) + ".o")
    cmd = [HIPCC, *HIP_FLAGS, "-c", src, "-o", obj]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"hipcc failed for {src}:\n{r.stdout}\n{r.stderr}")
    return obj


def _compile_bind() -> str:
    """serve_bind.cpp against the installed torch's headers (host code only)."""
    import sysconfig

    import torch
    from torch.utils import cpp_extension

    obj = os.path.join(BUILD, "serve_bind.o")
    cmd = ["g++", "-std=c++17", "-O2", "-fPIC", "-Wall", "-fvisibility=hidden", "-D__HIP_PLATFORM_AMD__", "-DUSE_ROCM",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}",
           *[a for d in [*cpp_extension.include_paths(), sysconfig.get_paths()["include"]] for a in ("-isystem", d)],
           "-c", os.path.join(CSRC, "serve_bind.cpp"), "-o", obj]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"g++ failed for serve_bind.cpp:\n{r.stdout}\n{r.stderr}")
    return obj


def _link_bind(obj: str) -> None:
    from torch.utils import cpp_extension

    tmp = BIND + ".tmp"
    dirs = cpp_extension.library_paths()
    cmd = ["g++", "-shared", "-o", tmp, obj, LIB, *[f"-L{d}" for d in dirs], "-ltorch_python", "-ltorch_cpu", "-lc10",
           "-Wl,-rpath,$ORIGIN"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, BIND)


def build(verbose: bool = False) -> str:
    os.makedirs(BUILD, exist_ok=True)
    srcs = sorted(glob.glob(os.path.join(CSRC, "*.hip")))
    with cf.ThreadPoolExecutor(max_workers=min(8, len(srcs) + 1)) as ex:
        bind = ex.submit(_compile_bind)
        objs = list(ex.map(_compile, srcs))
        bind = bind.result()
    tmp = LIB + ".tmp"
    cmd = [HIPCC, "--offload-arch=gfx950", "-shared", "-fPIC", "-Wl,-soname,libnrq.so", "-o", tmp, *objs]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, LIB)
    _link_bind(bind)
    if verbose:
        print(f"built {LIB}")
    return LIB


if __name__ == "__main__":
    build(verbose=True)
    sys.exit(0)
