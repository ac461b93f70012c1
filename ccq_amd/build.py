"""Build libccq_hip.so (all HIP sources, gfx950) in-tree with hipcc, and _ccq_torch.so (the PyTorch side of the operators
around the mixers, C++) beside it."""

from __future__ import annotations

import os
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
BUILD = os.path.join(HERE, "_build")
LIB = os.path.join(HERE, "libccq_hip.so")
SOURCES = ["ccq_abi.hip", "ccq_cwalk.hip", "ccq_gdn.hip", "ccq_gwalk.hip", "ccq_gla.hip", "ccq_decode.hip", "ccq_zclean.hip", "ccq_misc.hip", "ccq_cseg.hip", "ccq_prologue.hip",
           "ccq_linear.hip", "ccq_norm.hip", "ccq_logprobs.hip"]
TORCH_SOURCE = "ccq_torch.cpp"
TORCH_LIB = os.path.join(HERE, "_ccq_torch.so")
CXX = os.environ.get("CXX", "g++")
ROCM = os.environ.get("ROCM_PATH", "/opt/rocm")
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
ARCH = "gfx950"
FLAGS = [
    f"--offload-arch={ARCH}", "-O3", "-std=c++17", "-fPIC",
    # packed fp32 arithmetic is left to the compiler's scalar code paths
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-Wno-unused-result",
]


def _compile(src: str) -> str:
    obj = os.path.join(BUILD, src.replace(".hip", ".o"))
    cmd = [HIPCC, *FLAGS, "-c", os.path.join(CSRC, src), "-o", obj]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"hipcc failed for {src}:\n{r.stderr}")
    return obj


def _run(cmd, what: str) -> None:
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"{what} failed:\n{r.stderr}")


def _compile_torch() -> str:
    from torch.utils.cpp_extension import include_paths
    obj = os.path.join(BUILD, "ccq_torch.o")
    includes = [*include_paths(), sysconfig.get_paths()["include"], os.path.join(ROCM, "include")]
    _run([CXX, "-O2", "-std=c++17", "-fPIC", "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1",
          "-DTORCH_EXTENSION_NAME=_ccq_torch", *[a for d in includes for a in ("-isystem", d)], "-c",
          os.path.join(CSRC, TORCH_SOURCE), "-o", obj], f"{CXX} for {TORCH_SOURCE}")
    return obj


def _link_torch(obj: str) -> None:
    import torch
    tmp = TORCH_LIB + ".tmp"
    _run([CXX, "-shared", "-fPIC", "-o", tmp, obj, "-L" + HERE, "-l:" + os.path.basename(LIB), "-Wl,-rpath,$ORIGIN",
          "-L" + os.path.join(os.path.dirname(torch.__file__), "lib"), "-lc10", "-ltorch_cpu", "-ltorch",
          "-ltorch_python", "-lc10_hip", "-ltorch_hip"], f"link of {TORCH_LIB}")
    os.replace(tmp, TORCH_LIB)


def build(verbose: bool = True) -> str:
    os.makedirs(BUILD, exist_ok=True)
    with ThreadPoolExecutor(max_workers=min(8, len(SOURCES) + 1)) as ex:
        torch_obj = ex.submit(_compile_torch)
        objs = list(ex.map(_compile, SOURCES))
    tmp = LIB + ".tmp"
    cmd = [HIPCC, f"--offload-arch={ARCH}", "-shared", "-fPIC", "-o", tmp, *objs]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{r.stderr}")
    os.replace(tmp, LIB)
    _link_torch(torch_obj.result())
    if verbose:
        print(f"built {LIB} and {TORCH_LIB}")
    return LIB


if __name__ == "__main__":
    build()
    sys.exit(0)
