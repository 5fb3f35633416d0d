"""Build libptwm_mi355x.so in-tree with hipcc for gfx950, and the native
module of the MX operators' Python entry points.

Usage: ``python -m ptwm_amd.build`` (also called by ``__graft_entry__.build``).
Always recompiles every source: the caller asked for a build.
"""
from __future__ import annotations

import concurrent.futures as cf
import importlib.util
import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OBJ = os.path.join(HERE, "_build")
LIB = os.path.join(HERE, "libptwm_mi355x.so")
MX = os.path.join(HERE, "_mx.so")  # Python entry points of the MX operators
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")

SOURCES = ["transform.hip", "decode_exact.hip", "decode_sync.hip", "zstd_device.hip", "o1sac_device.hip", "huff_ilv.hip", "rans_ilv.hip", "ilv_host.hip", "rans_host.hip", "huffman_host.cpp", "code_tables.hip", "runtime.hip", "plane_ops.hip",
           "ref_encode.hip", "integrity.hip", "hash_host.hip", "xxh64_host.cpp", "container.cpp", "container_write.cpp", "blake3_host.cpp", "plan_parse.cpp",
           "mx_activations.hip", "mx_linear.hip", "mx_quantise.hip", "mx_matmul.hip", "mx_moe.hip", "abi.hip"]

CFLAGS = [
    "--offload-arch=gfx950",
    "-O3",
    "-std=c++17",
    "-fPIC",
    # packed-FP32 instructions are kept out of every kernel on purpose
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-Wall",
    "-Wno-unused-function",
]


def _compile(src: str) -> str:
    obj = os.path.join(OBJ, os.path.splitext(src)[0] + ".o")
    cmd = [HIPCC, *CFLAGS, "-c", os.path.join(CSRC, src), "-o", obj]
    r = subprocess.run(cmd, capture_output=True, text=True)
    noise = "is not a recognized feature for this target"
    err = "\n".join(l for l in (r.stderr or "").splitlines() if noise not in l)
    if r.returncode != 0:
        raise RuntimeError(f"hipcc failed for {src}:\n{err}")
    if err.strip():
        print(err, file=sys.stderr)
    return obj


def _compile_mx() -> str:
    """The Python entry points of the MX operators, host code against torch's headers."""
    import sysconfig

    import torch
    from torch.utils import cpp_extension

    obj = os.path.join(OBJ, "mx_python.o")
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-Wall", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}",
           *(f"-I{p}" for p in cpp_extension.include_paths()), f"-I{sysconfig.get_path('include')}",
           "-c", os.path.join(CSRC, "mx_python.cpp"), "-o", obj]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"g++ failed for mx_python.cpp:\n{r.stderr}")
    if r.stderr.strip():
        print(r.stderr, file=sys.stderr)
    return obj


def _link_mx(obj: str) -> None:
    from torch.utils import cpp_extension

    tmp = MX + ".tmp"
    libs = [f"-L{p}" for p in cpp_extension.library_paths()]
    cmd = ["g++", "-shared", "-o", tmp, obj, *libs, "-ltorch_python", "-ltorch_cpu", "-lc10", "-ldl"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link of the MX operators' module failed:\n{r.stderr}")
    os.replace(tmp, MX)


def build(verbose: bool = False) -> str:
    """Builds the library, and after it the module of the MX operators where torch is there to compile it against."""
    os.makedirs(OBJ, exist_ok=True)
    with_mx = importlib.util.find_spec("torch") is not None
    with cf.ThreadPoolExecutor(max_workers=min(8, len(SOURCES))) as ex:
        mx = ex.submit(_compile_mx) if with_mx else None
        objs = list(ex.map(_compile, SOURCES))
    tmp = LIB + ".tmp"
    cmd = [HIPCC, "--offload-arch=gfx950", "-shared", "-fPIC", "-o", tmp, *objs]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{r.stderr}")
    os.replace(tmp, LIB)
    if mx is not None:
        _link_mx(mx.result())
    else:
        if os.path.exists(MX):
            os.remove(MX)
        print("no torch: the Python entry points of the MX operators are not built", file=sys.stderr)
    if verbose:
        print(f"built {LIB}")
    return LIB


if __name__ == "__main__":
    build(verbose=True)
