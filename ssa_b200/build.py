"""Build the sm_100a kernel library `ssa_b200/libssa_b200.so` in-tree.

    python -m ssa_b200.build [--force]

Each .cu file is compiled by nvcc for `-gencode arch=compute_100a,code=sm_100a`
(in parallel), then linked into one shared library with the static CUDA
runtime. The library exports only the C ABI of include/ssa_b200.h. Then
`ssa_b200/_ssa_torch.so`, the Python module of the block cache's operators for
torch tensors (ssa_torch.cpp), is compiled against torch's headers and linked
to that library beside it.
"""
from __future__ import annotations

import argparse
import os
import shutil
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor

PKG = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG)
CSRC = os.path.join(PKG, "csrc")
OBJ_DIR = os.path.join(PKG, "_build")
LIB = os.path.join(PKG, "libssa_b200.so")
TORCH_LIB = os.path.join(PKG, "_ssa_torch.so")
SOURCES = ["ssa_graph.cu", "ssa_select_tc.cu", "ssa_hash_tc.cu", "ssa_select_rows.cu", "ssa_attn.cu", "ssa_cache.cu",
           "ssa_cache_attn.cu", "ssa_cache_prompt.cu", "ssa_capi.cu"]
HEADERS = ["ssa_common.cuh", "ssa_internal.h", "ssa_select_common.cuh", "ssa_tcgen05.cuh",
           "ssa_cache.cuh", "ssa_cache_attn.cuh"]
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=hidden",
         "--expt-relaxed-constexpr"]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", shutil.which("nvcc")):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found")


def _stale(target: str, deps) -> bool:
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


def build(force: bool = False, verbose: bool = False) -> str:
    os.makedirs(OBJ_DIR, exist_ok=True)
    pool = ThreadPoolExecutor(max_workers=1)
    ext = pool.submit(build_torch, force, verbose)  # beside the .cu files
    hdrs = [os.path.join(CSRC, h) for h in HEADERS] + [os.path.join(ROOT, "include", "ssa_b200.h")]
    jobs = []
    for src in SOURCES:
        s = os.path.join(CSRC, src)
        o = os.path.join(OBJ_DIR, src.replace(".cu", ".o"))
        if force or _stale(o, [s] + hdrs):
            jobs.append((s, o))

    def compile_one(job):
        s, o = job
        cmd = [nvcc()] + ARCH + FLAGS + ["-c", s, "-o", o + ".tmp"]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"nvcc failed for {s}:\n{r.stderr}")
        os.replace(o + ".tmp", o)
        if verbose:
            print("compiled", os.path.basename(s))

    with ThreadPoolExecutor(max_workers=len(jobs) or 1) as ex:
        list(ex.map(compile_one, jobs))
    objs = [os.path.join(OBJ_DIR, s.replace(".cu", ".o")) for s in SOURCES]
    if force or jobs or _stale(LIB, objs):
        tmp = LIB + f".tmp{os.getpid()}"
        cmd = [nvcc()] + ARCH + ["-shared", "-cudart", "static", "-o", tmp] + objs
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"link failed:\n{r.stderr}")
        os.replace(tmp, LIB)
        if verbose:
            print("linked", LIB)
    ext.result()
    pool.shutdown()
    return LIB


def build_torch(force: bool = False, verbose: bool = False) -> str:
    """_ssa_torch.so from ssa_torch.cpp. It resolves the C ABI at load time
    from the libssa_b200.so that ssa_b200._lib has loaded."""
    src = os.path.join(CSRC, "ssa_torch.cpp")
    if not (force or _stale(TORCH_LIB, [src, os.path.join(ROOT, "include", "ssa_b200.h")])):
        return TORCH_LIB
    import torch
    from torch.utils import cpp_extension as ext
    inc = [f"-I{p}" for p in ext.include_paths() + ["/usr/local/cuda/include", sysconfig.get_paths()["include"]]]
    lib = [f"-L{p}" for p in ext.library_paths()]
    tmp = TORCH_LIB + f".tmp{os.getpid()}"
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden", "-DTORCH_EXTENSION_NAME=_ssa_torch",
           "-DTORCH_API_INCLUDE_EXTENSION_H", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           *inc, src, "-o", tmp, *lib, "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_cuda", "-ltorch", "-ltorch_python"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"g++ failed for {src}:\n{r.stderr}")
    os.replace(tmp, TORCH_LIB)
    if verbose:
        print("linked", TORCH_LIB)
    return TORCH_LIB


def main(argv=None):
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    args = ap.parse_args(argv)
    print(build(force=args.force, verbose=True))


if __name__ == "__main__":
    sys.exit(main())
