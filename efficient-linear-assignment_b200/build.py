"""Build the in-tree CUDA library libela_auction.so for sm_100a.

Run ``python efficient-linear-assignment_b200/build.py`` (or
``__graft_entry__.build()``).  nvcc cross-compiles, so no GPU is needed.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys

PKG_DIR = os.path.dirname(os.path.abspath(__file__))
REPO_DIR = os.path.dirname(PKG_DIR)
CSRC = os.path.join(PKG_DIR, "csrc")
# every source of the library with the headers it includes (each is compiled to its own object)
SOURCES = {
    "ela_auction.cu": ["ela_implicit.cuh"],
    "ela_expert.cu": ["ela_expert.cuh"],
    "ela_expert_route.cu": ["ela_expert.cuh"],
    "ela_expert_4bit.cu": ["ela_expert.cuh", "ela_expert_mma.cuh", "ela_expert_stream.cuh", "ela_expert_4bit.cuh"],
    "ela_expert_linear.cu": ["ela_expert.cuh", "ela_expert_mma.cuh", "ela_expert_stream.cuh"],
}
OUT = os.path.join(PKG_DIR, "libela_auction.so")
INCLUDE = os.path.join(REPO_DIR, "include")

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-lineinfo", "-std=c++17",
    "-Xcompiler", "-fPIC",
    "--expt-relaxed-constexpr",
]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", shutil.which("nvcc")):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found")


OP_SOURCES = [os.path.join(CSRC, "ela_torch_op.cpp"), os.path.join(CSRC, "ela_expert_op.cpp")]
OP_OUT = os.path.join(PKG_DIR, "libela_torch_op.so")


def _headers() -> list[str]:
    return [os.path.join(INCLUDE, h) for h in sorted(os.listdir(INCLUDE)) if h.endswith(".h")]


def _newer(out: str, deps: list[str]) -> bool:
    return os.path.exists(out) and all(os.path.getmtime(out) >= os.path.getmtime(d) for d in deps)


def build_op(force: bool = False) -> str:
    """Compile the C++ torch operators (torch.ops.ela_native.*) over
    libela_auction.so, unless the library is newer than its sources."""
    if not force and _newer(OP_OUT, [*OP_SOURCES, OUT, *_headers()]):
        return OP_OUT
    import torch
    tdir = os.path.dirname(torch.__file__)
    abi = int(torch._C._GLIBCXX_USE_CXX11_ABI)
    cuda_inc = os.path.join(os.path.dirname(os.path.dirname(nvcc())), "include")
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared", f"-D_GLIBCXX_USE_CXX11_ABI={abi}",
           "-I", os.path.join(tdir, "include"), "-I", os.path.join(tdir, "include", "torch", "csrc", "api", "include"),
           "-I", cuda_inc, "-I", INCLUDE, *OP_SOURCES, "-o", OP_OUT + ".tmp", "-L", PKG_DIR, "-lela_auction",
           "-L", os.path.join(tdir, "lib"), "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_cuda", "-ltorch",
           # the shared C++ runtime that torch uses, by name: a compiler that links its own static copy
           # brings a second set of locale facets, and formatting a number in an error message then crashes
           "-nostdlib++", "-l:libstdc++.so.6", "-Wl,-rpath,$ORIGIN"]
    subprocess.run(cmd, check=True)
    os.replace(OP_OUT + ".tmp", OP_OUT)
    return OP_OUT


def build(force: bool = False, verbose: bool = False) -> str:
    """Compile libela_auction.so unless it is newer than its sources (the
    sources whose object is out of date are compiled side by side)."""
    objects, running = [], []
    for src, includes in SOURCES.items():
        obj = os.path.join(CSRC, src[:-3] + ".o")
        objects.append(obj)
        if not force and _newer(obj, [os.path.join(CSRC, f) for f in [src, *includes]] + _headers()):
            continue
        cmd = [nvcc(), *NVCC_FLAGS, "-c", "-I", INCLUDE, "-o", obj + ".tmp", os.path.join(CSRC, src)]
        if verbose:
            cmd.insert(1, "-Xptxas=-v")
        running.append((obj, cmd, subprocess.Popen(cmd)))
    for obj, cmd, p in running:
        if p.wait() != 0:
            raise subprocess.CalledProcessError(p.returncode, cmd)
        os.replace(obj + ".tmp", obj)
    if force or not _newer(OUT, objects):
        subprocess.run([nvcc(), *NVCC_FLAGS, "-shared", "-o", OUT + ".tmp", *objects], check=True)
        os.replace(OUT + ".tmp", OUT)
    return OUT


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
    print(build_op(force="--force" in sys.argv))
