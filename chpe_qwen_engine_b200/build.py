"""Build the native libraries in-tree.

* libchpe.so        -- the product: C ABI + CUDA kernels for sm_100a (nvcc)
* libchpe_synth.so  -- deterministic synthetic archive generator (gcc)
* _ops.so           -- the batched decode operators on torch tensors, a CPython
                       module over libchpe.so (g++, torch's headers; left out
                       where torch is missing, rebuilt when torch changes)
* chpe_fwd          -- the command-line front end over libchpe.so (the
                       reference's chpe_fwd contract)

Usage: python -m chpe_qwen_engine_b200.build [--force]
"""
from __future__ import annotations

import importlib.metadata
import importlib.util
import os
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

PKG = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(PKG, "csrc")
ROOT = os.path.dirname(PKG)
LIBCHPE = os.path.join(PKG, "libchpe.so")
LIBSYNTH = os.path.join(PKG, "libchpe_synth.so")
CHPE_FWD = os.path.join(PKG, "chpe_fwd")
OPS = os.path.join(PKG, "_ops.so")
OPS_TAG = os.path.join(PKG, "_build", "_ops.tag")  # what _ops.so was built against

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-lineinfo", "-std=c++17",
    "-Xcompiler", "-fPIC", "-Xcompiler", "-Wall",
    "--expt-relaxed-constexpr",
    "-I", CSRC, "-I", os.path.join(ROOT, "include"),
]

ENGINE_SRCS = ["engine.cu", "engine_verify.cu", "attention_noalloc.cu", "deltanet.cu", "chpe_convert.cu", "tc_probe.cu",
               "qk_rope.cu", "attention_paged.cu", "logits.cu",
               "chpe_c_api.cpp", "chpe_maps.c"]
ENGINE_DEPS = ENGINE_SRCS + ["engine.h", "engine_types.h", "gemv.cuh", "attention.cuh",
                             "aux_kernels.cuh", "gemv_tma.cuh", "gemv_flat_tma.cuh", "gemv_rowblk.cuh", "device_common.cuh", "chpe_maps.h",
                             "tc_common.cuh", "bgemm_tc.cuh", "serve_common.h", "buffer_rows.h",
                             "qwen3b_cell_map.inc", "../../include/chpe.h"]
SYNTH_SRCS = ["chpe_synth.c", "chpe_maps.c"]
SYNTH_DEPS = SYNTH_SRCS + ["chpe_synth.h", "chpe_maps.h", "qwen3b_cell_map.inc"]


def _nvcc() -> str:
    for c in ("nvcc", "/usr/local/cuda/bin/nvcc"):
        p = shutil.which(c) or (c if os.path.exists(c) else None)
        if p:
            return p
    raise RuntimeError("nvcc not found")


def _stale(target: str, deps: list[str]) -> bool:
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(os.path.join(CSRC, d)) > t for d in deps)


def build_synth(force: bool = False) -> str:
    if force or _stale(LIBSYNTH, SYNTH_DEPS):
        cmd = ["gcc", "-O2", "-fPIC", "-shared", "-pthread", "-Wall", "-Wextra", "-o", LIBSYNTH]
        cmd += [os.path.join(CSRC, s) for s in SYNTH_SRCS]
        subprocess.run(cmd, check=True)
    return LIBSYNTH


def build_engine(force: bool = False) -> str:
    if force or _stale(LIBCHPE, ENGINE_DEPS):
        objdir = os.path.join(PKG, "_build")
        os.makedirs(objdir, exist_ok=True)
        nvcc = _nvcc()

        def compile_one(s: str) -> str:
            o = os.path.join(objdir, os.path.splitext(s)[0] + ".o")
            src = os.path.join(CSRC, s)
            if s.endswith(".c"):
                cmd = ["gcc", "-O2", "-fPIC", "-c", src, "-o", o, "-I", CSRC]
            else:
                cmd = [nvcc] + NVCC_FLAGS + ["-c", src, "-o", o]
            subprocess.run(cmd, check=True)
            return o

        with ThreadPoolExecutor(max_workers=max(1, min(8, os.cpu_count() or 1))) as pool:
            objs = list(pool.map(compile_one, ENGINE_SRCS))
        cmd = [nvcc, "-gencode", "arch=compute_100a,code=sm_100a", "-shared", "-o", LIBCHPE] + objs
        subprocess.run(cmd, check=True)
    return LIBCHPE


def build_cli(force: bool = False) -> str:
    """chpe_fwd, linked against the in-tree libchpe.so (found through $ORIGIN)."""
    if force or _stale(CHPE_FWD, ["chpe_fwd.cpp", "../../include/chpe.h"]) or (
            os.path.exists(CHPE_FWD) and os.path.getmtime(LIBCHPE) > os.path.getmtime(CHPE_FWD)):
        cmd = [_nvcc(), "-gencode", "arch=compute_100a,code=sm_100a", "-O2", "-std=c++17", "-o", CHPE_FWD, os.path.join(CSRC, "chpe_fwd.cpp"),
               "-I", os.path.join(ROOT, "include"), "-L", PKG, "-lchpe", "-Xlinker", "-rpath=$ORIGIN"]
        subprocess.run(cmd, check=True)
    return CHPE_FWD


def _torch_tag() -> str:
    """What _ops.so is built against: torch, Python; "" where torch, or its CUDA part, is missing."""
    spec = importlib.util.find_spec("torch")
    root = os.path.dirname(spec.origin) if spec and spec.origin else ""
    if not root or not os.path.exists(os.path.join(root, "lib", "libc10_cuda.so")):
        return ""
    return f"{importlib.metadata.version('torch')} {sys.implementation.cache_tag} {root}"


def build_ops(force: bool = False) -> str | None:
    """_ops.so, linked against the in-tree libchpe.so (found through $ORIGIN)
    and the installed torch; None where there is none (the engine, its ctypes
    interface and the command line do without)."""
    tag = _torch_tag()
    if not tag:
        print("_ops.so is not built: no torch with CUDA", file=sys.stderr)
        return None
    try:
        with open(OPS_TAG) as f:
            same = f.read() == tag
    except OSError:
        same = False
    if force or not same or _stale(OPS, ["ops_torch.cpp", "../../include/chpe.h"]):
        import sysconfig

        import torch
        from torch.utils.cpp_extension import include_paths
        lib = os.path.join(os.path.dirname(torch.__file__), "lib")
        cuda = os.path.join(os.path.dirname(os.path.dirname(os.path.realpath(_nvcc()))), "include")
        cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-Wall", "-o", OPS, os.path.join(CSRC, "ops_torch.cpp"),
               f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}",
               "-I", os.path.join(ROOT, "include"), "-isystem", sysconfig.get_paths()["include"], "-isystem", cuda]
        for p in include_paths():
            cmd += ["-isystem", p]
        cmd += ["-L", PKG, "-lchpe", "-Wl,-rpath,$ORIGIN", "-L", lib, "-lc10", "-lc10_cuda", "-ltorch", "-ltorch_cpu",
                "-ltorch_python"]
        subprocess.run(cmd, check=True)
        os.makedirs(os.path.dirname(OPS_TAG), exist_ok=True)
        with open(OPS_TAG, "w") as f:
            f.write(tag)
    return OPS


def build_all(force: bool = False) -> list[str]:
    return [p for p in (build_synth(force), build_engine(force), build_cli(force), build_ops(force)) if p]


if __name__ == "__main__":
    print("built", *build_all(force="--force" in sys.argv))
