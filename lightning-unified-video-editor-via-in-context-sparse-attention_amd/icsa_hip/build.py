"""Build ``libicsa.so`` (gfx950) from ``../csrc`` with hipcc, and ``_autograd.so`` (host code) with g++.

Every HIP source is compiled to an object in ``csrc/_build`` (in parallel), then linked
into ``icsa_hip/libicsa.so`` next to this file.  The link goes to a
temporary name first and is renamed into place, so a concurrent loader never sees a
half-written library.  ``_autograd.so`` (the autograd nodes of ``train.py``) is built beside it against the
installed torch.  Where that cannot be (no g++, no headers) the command fails, after ``libicsa.so`` is in place: the C library needs hipcc alone.
Run ``python -m icsa_hip.build`` or call :func:`build_library`.
"""
from __future__ import annotations

import os
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

PKG_DIR = os.path.dirname(os.path.abspath(__file__))
CSRC_DIR = os.path.join(os.path.dirname(PKG_DIR), "csrc")
BUILD_DIR = os.path.join(CSRC_DIR, "_build")
LIB_PATH = os.path.join(PKG_DIR, "libicsa.so")
NODES_PATH = os.path.join(PKG_DIR, "_autograd.so")

SOURCES = ["pool.hip", "compressed.hip", "newkv.hip", "gather.hip", "flash_attn.hip", "sparse_attn.hip", "sparse_bwd.hip",
           "wan_qk.hip", "wan_block.hip", "mx_quant.hip", "mx_gemm.hip", "mx_rows.hip", "masked_attn.hip",
           "attn_bwd.hip", "norm.hip", "rotary.hip", "api.hip"]

HIP_FLAGS = [
    "--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC",
    # packed fp32 VALU forms are kept out of every kernel
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-Wno-unused-command-line-argument",
]

# Per-source additions.  The flash kernel is scheduled with LLVM's memory-clause strategy:
# in alternating runs its stage took 19.84-19.85 ms against 19.90-19.98 ms with the
# default strategy on one box (the dense baseline 70.2-70.4 against 70.7-70.8 ms) and
# 19.73-19.75 against 19.83-19.89 ms on another, with the same 196 registers and no
# spills.  The max-ilp and iterative-ilp strategies were slower (20.0-20.2 and
# 20.7-21.0 ms), and the other kernels gained nothing from any of them.
EXTRA_FLAGS = {
    "flash_attn.hip": ["-mllvm", "-amdgpu-sched-strategy=max-memory-clause"],
}


def _hipcc() -> str:
    for cand in (os.environ.get("HIPCC"), "/opt/rocm/bin/hipcc"):
        if cand and os.path.exists(cand):
            return cand
    return "hipcc"


def _run(cmd, verbose):
    if verbose:
        print(" ".join(cmd), flush=True)
    res = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    out = "\n".join(l for l in res.stdout.splitlines() if "packed-fp32-ops" not in l and
                    "is not a recognized feature" not in l)
    if res.returncode != 0:
        raise RuntimeError(f"command failed ({res.returncode}): {' '.join(cmd)}\n{out}")
    if verbose and out.strip():
        print(out, flush=True)


def _build_nodes(verbose: bool) -> None:
    import sysconfig

    import torch
    from torch.utils.cpp_extension import include_paths

    lib = os.path.join(os.path.dirname(torch.__file__), "lib")
    tmp = NODES_PATH + f".tmp{os.getpid()}"
    # torch's headers ask for the platform's name; this file itself holds no device code
    _run([os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared", "-DTORCH_API_INCLUDE_EXTENSION_H",
          f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1",
          *(x for p in include_paths() for x in ("-isystem", p)), "-isystem", "/opt/rocm/include", "-isystem",
          sysconfig.get_paths()["include"], os.path.join(CSRC_DIR, "autograd.cpp"), "-o", tmp, f"-L{lib}",
          "-lc10", "-lc10_hip", "-ltorch_cpu", "-ltorch", "-ltorch_python"], verbose)
    os.replace(tmp, NODES_PATH)


def build_library(verbose: bool = False, jobs: int = 8) -> str:
    """Compile every HIP source for gfx950 and link libicsa.so; returns its path."""
    os.makedirs(BUILD_DIR, exist_ok=True)
    hipcc = _hipcc()
    inc = ["-I", CSRC_DIR, "-I", os.path.join(os.path.dirname(os.path.dirname(PKG_DIR)), "include")]

    def compile_one(src):
        obj = os.path.join(BUILD_DIR, src.replace(".hip", ".o"))
        _run([hipcc, *HIP_FLAGS, *EXTRA_FLAGS.get(src, []), *inc, "-c", os.path.join(CSRC_DIR, src), "-o", obj],
             verbose)
        return obj

    with ThreadPoolExecutor(max_workers=max(1, min(jobs, len(SOURCES) + 1))) as ex:
        nodes = ex.submit(_build_nodes, verbose)          # the longest one first
        objs = list(ex.map(compile_one, SOURCES))
        tmp = LIB_PATH + f".tmp{os.getpid()}"
        _run([hipcc, "--offload-arch=gfx950", "-shared", "-fPIC", "-o", tmp, *objs], verbose)
        os.replace(tmp, LIB_PATH)
        nodes.result()                                    # the library is in place, whatever the host compiler says
    return LIB_PATH


if __name__ == "__main__":
    path = build_library(verbose="-v" in sys.argv)
    print(path)
